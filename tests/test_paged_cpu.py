"""Refusals of the paged cache's C ABI, without a device.

tla_paged_create checks everything before it touches the context, so a zeroed
block stands in for one here; a call that passed the checks would be a failure
of these tests. The reference's own forms are checked against small cases that
are written out."""
import ctypes

import pytest
import torch

from tests import paged_ref as ref

INVALID, UNSUPPORTED, ROTARY = -1, -9, -8


def create(pkg, flags=0, head_dim=64, heads=4, kv_heads=2, key=1 << 20, value=1 << 21, bounds=0, pages=8, page=16,
           strides=None, ctx=True, **more):
    from three_llm_b200 import _abi

    cfg = _abi.AttnConfig()
    cfg.head_count, cfg.kv_head_count, cfg.head_dim, cfg.max_tokens, cfg.max_batch = heads, kv_heads, head_dim, 128, 4
    cfg.rotary_dim, cfg.rope_pair_count = -1, -1
    cfg.rope_theta, cfg.flags = 10000.0, flags
    for k, v in more.items():
        setattr(cfg, k, v)
    pool = _abi.PagePool()
    pool.key, pool.value, pool.bounds = key, value, bounds
    pool.page_stride, pool.head_stride, pool.slot_stride = strides or (kv_heads * page * head_dim, page * head_dim,
                                                                       head_dim)
    pool.page_count, pool.page_size = pages, page
    block, out = ctypes.create_string_buffer(4096), ctypes.c_void_p(1)
    rc = pkg.lib().tla_paged_create(ctypes.cast(block, ctypes.c_void_p) if ctx else None, ctypes.byref(cfg),
                                    ctypes.byref(pool), None, None, ctypes.byref(out))
    assert rc != 0 and not out.value
    return rc


@pytest.mark.parametrize("args,code", [
    (dict(ctx=False), INVALID),
    (dict(key=0), INVALID),
    (dict(value=0), INVALID),
    (dict(value=1 << 20), INVALID),                        # key and value in the same memory
    (dict(key=(1 << 20) + 1), INVALID),                    # half an element
    (dict(bounds=8), INVALID),                             # not 16-byte aligned
    (dict(pages=0), INVALID),
    (dict(page=0, strides=(64, 64, 64)), INVALID),
    (dict(page=24), INVALID),                              # not a power of two
    (dict(page=2048), INVALID),
    (dict(strides=(2048, 1024, 63)), INVALID),             # slots overlap
    (dict(strides=(2048, 0, 64)), INVALID),                # broadcast heads
    (dict(strides=(2047, 1024, 64)), INVALID),             # pages overlap
    (dict(strides=(-2048, 1024, 64)), INVALID),
    (dict(strides=(1 << 62, 1024, 64)), INVALID),
    (dict(heads=5), UNSUPPORTED),                          # heads do not divide
    (dict(heads=65536), UNSUPPORTED),
    (dict(head_dim=257), UNSUPPORTED),
    (dict(kv_heads=8), INVALID),                           # more kv heads than heads
    (dict(flags=(1 << 2) | (1 << 4)), INVALID),            # two I/O types
    (dict(flags=(1 << 3) | (1 << 5)), INVALID),            # two page types
    (dict(flags=1 << 4), UNSUPPORTED),                     # bfloat16 over float16 pages
    (dict(flags=1 << 5), UNSUPPORTED),
    (dict(flags=1 << 3), UNSUPPORTED),                     # float16 over float32 pages
    (dict(max_tokens=0), INVALID),
    (dict(max_batch=0), INVALID),
    (dict(sliding_window=-1), INVALID),
    (dict(rotary_dim=3), ROTARY),
    (dict(rope_theta=0.5), -3),
])
def test_create_refuses(pkg, args, code):
    assert create(pkg, **args) == code


def test_calls_refuse_a_missing_layer(pkg):
    lib = pkg.lib()
    size = ctypes.c_size_t()
    assert lib.tla_paged_workspace(None, 1, 1, 0, ctypes.byref(size), ctypes.byref(size)) == INVALID
    assert lib.tla_paged_append(None, 16, 16, None, 16, 1, 1, 1, 16, None) == INVALID
    assert lib.tla_paged_decode(None, 16, 16, 16, 1, None, 0, None, 16, 1, 16, 16, None) == INVALID
    assert lib.tla_paged_select(None, 16, 16, 16, 1, 0, 0, 16, 1, 1, 16, 16, None) == INVALID
    assert lib.tla_paged_destroy(None) == 0


def test_contiguous_layers_refuse_bfloat16(pkg):
    from three_llm_b200 import _abi

    cfg = _abi.AttnConfig()
    cfg.head_count, cfg.kv_head_count, cfg.head_dim, cfg.max_tokens, cfg.max_batch = 4, 2, 64, 128, 4
    block, out = ctypes.create_string_buffer(4096), ctypes.c_void_p()
    for flag in (_abi.FLAG_IO_BF16, _abi.FLAG_CACHE_BF16):
        cfg.flags = flag
        assert pkg.lib().tla_layer_create(ctypes.cast(block, ctypes.c_void_p), ctypes.byref(cfg), None, None,
                                          ctypes.byref(out)) == UNSUPPORTED
        assert pkg.lib().tla_decode_noalloc(ctypes.byref(cfg), 16, 16, None, None, 16, 16, None, 16, None, 1,
                                            None) == UNSUPPORTED


def test_status_string_names_the_page(pkg):
    assert "page" in pkg.lib().tla_status_string(-18).decode()


def test_reference_leaves_bad_pages_out():
    """A table entry outside the pool takes its tokens out of the attention, and out of the selection."""
    g = torch.Generator().manual_seed(3)
    keys, values = (torch.randn(4, 1, 2, 4, generator=g) for _ in range(2))
    q = torch.randn(2, 4, generator=g)
    got, _ = ref.attend(q, keys, values, [1, 9, 2], 5, 2, 0.5, out_type=torch.float32, kept=torch.float32)
    rows_k = torch.cat((keys[1, 0], keys[2, 0])).double()
    rows_v = torch.cat((values[1, 0], values[2, 0])).double()
    exp = torch.softmax(q.double() @ rows_k.t() * 0.5, -1) @ rows_v
    assert torch.allclose(got, exp, atol=1e-12)
    bounds = torch.stack((keys.amin(2), keys.amax(2)), 2)
    assert ref.select(q, bounds, [1, 9, 2, 0, 3], 9, 2, 4, 1, 1) == [[0, 2, 3, 4]]
    assert ref.select(q, bounds, [1, -1, 2], -1, 2, 2) == [[-1, -1]]


def test_reference_attends_to_nothing_as_zeros():
    keys = torch.zeros(1, 1, 2, 4)
    out, tol = ref.attend(torch.ones(1, 4), keys, keys, [0], -1, 2, 1.0)
    assert not out.any() and (tol > 0).all()
    out, _ = ref.attend(torch.ones(1, 4), keys, keys + 1, [5], 1, 2, 1.0)
    assert not out.any()
