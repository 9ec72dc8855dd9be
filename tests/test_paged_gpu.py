"""GPU parity of the paged cache (PagedAttention through the C ABI) against the
64-bit forms of tests/paged_ref.py. Every slot that holds no token of a
sequence is NaN, and the tables' unused entries name no page, so a read of
either shows. Error bounds come with the reference's outputs; they count each
rounding, and are derived there."""
import ctypes
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
#: (activations, pages)
PAIRS = [("fp16", "fp16"), ("bf16", "bf16"), ("fp32", "fp16"), ("fp32", "bf16"), ("fp32", "fp32")]


class World:
    """A pool with the sequences' tokens in scattered pages, on the host and on the device."""

    def __init__(self, lengths, hk, d, page, kept, layout="HND", seed=0, spare=3, extra_width=1, room=0):
        g = torch.Generator().manual_seed(seed)
        self.g, self.page, self.layout, self.kept, self.lengths = g, page, layout, TYPES[kept], lengths
        held = [-(-(max(n, 0) + room) // page) for n in lengths]
        total = sum(held) + spare
        order = torch.randperm(total, generator=g).tolist()
        self.width = max(max(held), 1) + extra_width
        self.table, at = [], 0
        for n in held:
            self.table.append(order[at:at + n] + [-7] * (self.width - n))
            at += n
        self.keys = torch.full((total, hk, page, d), float("nan"), dtype=self.kept)
        self.values = self.keys.clone()
        self.bounds = torch.full((total, hk, 2, d), float("nan"), dtype=self.kept)
        for b, n in enumerate(lengths):
            for i in range(-(-n // page) if n > 0 else 0):
                m = min(page, n - i * page)
                p = self.table[b][i]
                self.keys[p, :, :m] = torch.randn(hk, m, d, generator=g).to(self.kept)
                self.values[p, :, :m] = torch.randn(hk, m, d, generator=g).to(self.kept)
                self.bounds[p, :, 0] = self.keys[p, :, :m].amin(1)
                self.bounds[p, :, 1] = self.keys[p, :, :m].amax(1)

    def device_pool(self, cuda):
        def put(t):
            t = t.to(cuda)
            return t if self.layout == "HND" else t.transpose(1, 2).contiguous()

        return put(self.keys), put(self.values), self.bounds.to(cuda)

    def device_table(self, cuda):
        return torch.tensor(self.table, dtype=torch.int32, device=cuda)

    def normal(self, *shape, dtype):
        return torch.randn(*shape, generator=self.g).to(dtype)


def by_head(t, layout):
    return t if layout == "HND" else t.transpose(1, 2)


def ints(v, cuda):
    return torch.tensor(v, dtype=torch.int32, device=cuda)


def close(got, exp, tol, what=""):
    got = got.double().cpu().reshape(exp.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - exp).abs()
    assert (off <= tol).all(), f"{what}: {(off > tol).sum()} of {off.numel()} off, worst by {(off - tol).max():.3e} over {tol.max():.3e}"


def make(pkg, cuda, w, hq, hk, d, io, bounds=True, **options):
    k, v, bd = w.device_pool(cuda)
    o = {"headDim": d, "kvHeadCount": hk, "dtype": TYPES[io], "pageLayout": w.layout, **options}
    layer = pkg.PagedAttention(hq * d, hq, w.width * w.page, k, v, o, key_bounds=bd if bounds else None)
    return layer, k, v, bd


# ---------------------------------------------------------------- decode
LENGTHS = [1, 2, 15, 16, 17, 63, 64, 65, 128, 129, 200, 511]
SHAPES = [(8, 2, 64), (14, 2, 64), (32, 8, 128), (16, 1, 128), (4, 4, 64), (40, 2, 64)]


def check_decode(pkg, cuda, lengths, hq, hk, d, page, io, kept, layout="HND", window=0, gated=False, listed=None,
                 scale=None, seed=0, extra_width=1):
    w = World(lengths, hk, d, page, kept, layout, seed=seed, extra_width=extra_width)
    options = {"slidingWindow": window}
    if scale is not None:
        options["attnScale"] = scale
    layer, *_ = make(pkg, cuda, w, hq, hk, d, io, **options)
    b = len(lengths)
    q = w.normal(b, hq, d, dtype=TYPES[io])
    gate = w.normal(b, hq * d, dtype=TYPES[io]) if gated else None
    pages, count = None, 0
    if listed is not None:
        count = max(len(x) for seq in listed for x in seq)
        pages = ints([[x + [-1] * (count - len(x)) for x in seq] for seq in listed], cuda)
    out = layer.decode(q.view(b, -1).to(cuda), ints([n - 1 for n in lengths], cuda), w.device_table(cuda), pages=pages,
                       gate=None if gate is None else gate.to(cuda))
    assert layer.context.error() == 0
    for i, n in enumerate(lengths):
        exp, tol = ref.attend(q[i], w.keys, w.values, w.table[i], n - 1, page, d ** -0.5 if scale is None else scale,
                              window, None if listed is None else listed[i], None if gate is None else gate[i],
                              TYPES[io], w.kept)
        close(out[i], exp, tol, f"sequence {i} of {n}")


@pytest.mark.parametrize("io,kept", PAIRS)
@pytest.mark.parametrize("hq,hk,d", SHAPES)
def test_decode_shapes_and_types(pkg, cuda, hq, hk, d, io, kept):
    check_decode(pkg, cuda, LENGTHS, hq, hk, d, 16, io, kept)


@pytest.mark.parametrize("page", [1, 8, 16, 32, 64, 128, 1024])
@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("d", [64, 128])
def test_decode_page_sizes_and_layouts(pkg, cuda, page, layout, d):
    check_decode(pkg, cuda, LENGTHS, 8, 2, d, page, "fp16", "fp16", layout)


@pytest.mark.parametrize("d", [2, 8, 80, 96, 256])
@pytest.mark.parametrize("io,kept", [("fp16", "fp16"), ("fp32", "fp32")])
def test_decode_other_head_dims(pkg, cuda, d, io, kept):
    check_decode(pkg, cuda, [1, 33, 130], 6, 2, d, 16, io, kept)


@pytest.mark.parametrize("d", [8, 24, 64, 80, 128, 200, 256])
@pytest.mark.parametrize("io,kept,page", [("fp32", "fp32", 16), ("fp32", "fp32", 1), ("fp32", "bf16", 64),
                                          ("bf16", "bf16", 4), ("fp16", "fp16", 8)])
def test_decode_rows(pkg, cuda, d, io, kept, page):
    """What goes row by row: float32 pages, float32 over bfloat16 pages, small pages."""
    check_decode(pkg, cuda, [1, 17, 64, 300, 0, 1000], 6, 2, d, page, io, kept, gated=True)
    check_decode(pkg, cuda, [77, 500], 10, 1, d, page, io, kept, layout="NHD", window=90)
    if page > 1:
        check_decode(pkg, cuda, [70, 200], 4, 2, d, page, io, kept,
                     listed=[[[0, 1], [0, 2, 3]], [[1], [0, 2, 199 // page]]] if page < 64 else [[[0, 1], [1]], [[0, 3], [2]]])


@pytest.mark.parametrize("d,io,kept,page,wide", [
    (64, "fp16", "fp16", 16, 1), (128, "bf16", "bf16", 64, 1), (256, "fp32", "fp16", 16, 1), (64, "fp16", "fp16", 16, 9000),
    (128, "fp32", "fp16", 16, 9000), (64, "fp32", "fp32", 16, 1), (100, "fp16", "fp16", 16, 1)])
def test_decode_nan_among_the_tokens(pkg, cuda, d, io, kept, page, wide):
    """A NaN in a key or value that takes part shows in the heads that read it, also where it is the only token."""
    lengths = [1, 40, 700, 1, 700]
    w = World(lengths, 2, d, page, kept, extra_width=wide)
    at = [w.table[i][n] for i, n in ((0, 0), (1, 37 // page), (2, 650 // page))]
    w.keys[at[0], 0, 0, d - 1] = float("nan")
    w.keys[at[1], 1, 37 % page, 0] = float("nan")
    w.values[at[2], 1, 650 % page] = float("nan")
    layer, *_ = make(pkg, cuda, w, 6, 2, d, io)
    out = layer.decode(w.normal(5, 6 * d, dtype=TYPES[io]).to(cuda), ints([n - 1 for n in lengths], cuda),
                       w.device_table(cuda))
    bad = out.view(5, 2, 3 * d).isnan().cpu()
    assert bad[0, 0].all() and bad[1, 1].all() and bad[2, 1].all() and int(bad.sum()) == 9 * d


@pytest.mark.parametrize("d", [8, 24, 72, 80, 96, 136, 200, 256])
@pytest.mark.parametrize("io,kept", [("fp16", "fp16"), ("bf16", "bf16"), ("fp32", "fp16")])
@pytest.mark.parametrize("wide", [1, 9000])
def test_decode_widths_between(pkg, cuda, d, io, kept, wide):
    """head_dims that the kernels built for 64, 128 and 256 take with zero columns, in clusters and in shares."""
    check_decode(pkg, cuda, [1, 17, 64, 300, 0, 1000], 6, 2, d, 32, io, kept, gated=True, extra_width=wide)
    check_decode(pkg, cuda, [77, 500], 20, 2, d, 16, io, kept, layout="NHD", window=90, extra_width=wide)


@pytest.mark.parametrize("window", [1, 5, 16, 64, 100, 10000])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("io,kept", [("fp16", "fp16"), ("bf16", "bf16"), ("fp32", "fp16")])
def test_decode_window_gate_and_scale(pkg, cuda, window, page, io, kept):
    check_decode(pkg, cuda, LENGTHS, 14, 2, 64, page, io, kept, window=window, gated=True, scale=0.2)


@pytest.mark.parametrize("io,kept", PAIRS)
@pytest.mark.parametrize("lengths", [[3000], [1, 2999, 700], [0, 5, 0, 900, 0]])
@pytest.mark.parametrize("d", [64, 128])
def test_decode_split_over_length_and_empty_rows(pkg, cuda, io, kept, lengths, d):
    """One long sequence is cut over many blocks; a row without a sequence (position -1) is zeros."""
    check_decode(pkg, cuda, lengths, 8, 2, d, 32, io, kept, seed=1)


WIDE = 40000  # table entries past the sequences' own: their capacity has the pairs' tiles cut into shares


@pytest.mark.parametrize("io,kept", PAIRS)
@pytest.mark.parametrize("hq,hk,d", SHAPES)
def test_decode_in_shares_shapes_and_types(pkg, cuda, hq, hk, d, io, kept):
    check_decode(pkg, cuda, LENGTHS + [0, 900], hq, hk, d, 16, io, kept, extra_width=WIDE)


@pytest.mark.parametrize("io,kept", [("fp16", "fp16"), ("bf16", "bf16"), ("fp32", "fp16")])
@pytest.mark.parametrize("lengths", [[5000], [1], [0], [0, 0], [1, 2999, 700], [0, 5, 0, 900, 0], [64] * 40,
                                     [1 + (i * 37) % 90 for i in range(301)]])
@pytest.mark.parametrize("d", [64, 128])
def test_decode_in_shares(pkg, cuda, io, kept, lengths, d):
    """Pairs held by one CTA and by many, empty rows, more pairs than CTAs and fewer; then with gates."""
    check_decode(pkg, cuda, lengths, 8, 2, d, 32, io, kept, seed=2, extra_width=WIDE // 2)
    check_decode(pkg, cuda, lengths[:40], 8, 2, d, 128, io, kept, layout="NHD", gated=True, extra_width=WIDE // 8)


def test_decode_listed_pages_in_shares(pkg, cuda):
    """Lists long enough for shares, most of them ending early."""
    lengths = [700, 16, 5000, 90]
    listed = [[list(range(0, 44, 3)), [43]], [[0], []], [list(range(1, 313)), [5, 6, 7, 100]], [[0, 2], [1, 5]]]
    count = 3000
    w = World(lengths, 2, 64, 16, "fp16", extra_width=WIDE)
    layer, *_ = make(pkg, cuda, w, 8, 2, 64, "fp16")
    q = w.normal(4, 8, 64, dtype=torch.float16)
    pages = ints([[x + [-1] * (count - len(x)) for x in seq] for seq in listed], cuda)
    out = layer.decode(q.view(4, -1).to(cuda), ints([n - 1 for n in lengths], cuda), w.device_table(cuda), pages=pages)
    assert layer.context.error() == 0
    for i, n in enumerate(lengths):
        exp, tol = ref.attend(q[i], w.keys, w.values, w.table[i], n - 1, 16, 0.125, listed=listed[i])
        close(out[i], exp, tol)


@pytest.mark.parametrize("wide", [0, WIDE])
def test_decode_faults_leave_the_other_rows(pkg, cuda, wide):
    """A page outside the pool in the middle of a long sequence, a position past the capacity, a row without
    a sequence and a good one, in one call."""
    w = World([3000, 3000, 0, 2000], 2, 128, 16, "fp16", extra_width=wide)
    layer, *_ = make(pkg, cuda, w, 8, 2, 128, "fp16")
    q = w.normal(4, 8, 128, dtype=torch.float16)
    table = [list(r) for r in w.table]
    table[0][77] = -5
    positions = [2999, w.width * 16, -1, 1999]
    out = layer.decode(q.view(4, -1).to(cuda), ints(positions, cuda), ints(table, cuda))
    assert layer.context.error() in (-12, -18)
    assert not out[1].any() and not out[2].any()
    for i in (0, 3):
        exp, tol = ref.attend(q[i], w.keys, w.values, table[i], positions[i], 16, 128 ** -0.5)
        close(out[i], exp, tol)


@pytest.mark.parametrize("hq,hk", [(1, 1), (3, 1), (16, 16), (64, 8), (8, 8), (33, 1), (128, 2)])
@pytest.mark.parametrize("wide", [0, WIDE])
def test_decode_head_groups(pkg, cuda, hq, hk, wide):
    check_decode(pkg, cuda, [1, 100, 333], hq, hk, 64, 16, "fp16", "fp16", extra_width=wide)
    check_decode(pkg, cuda, [77, 10], hq, hk, 128, 16, "fp32", "fp16", extra_width=wide)


def test_decode_many_sequences(pkg, cuda):
    check_decode(pkg, cuda, [1 + (i * 37) % 90 for i in range(301)], 4, 2, 64, 16, "fp16", "fp16")


@pytest.mark.parametrize("page", [8, 16, 64, 256])
@pytest.mark.parametrize("io,kept", [("fp16", "fp16"), ("bf16", "bf16"), ("fp32", "fp16")])
def test_decode_listed_pages(pkg, cuda, page, io, kept):
    """Lists of different lengths per kv head, empty ones among them; the last page is partly filled."""
    lengths = [7 * page - 3, page, 3 * page + 1, 5]
    listed = [[[0, 2, 3, 6], [6]], [[0], []], [[1, 3], [0, 1, 2, 3]], [[], []]]
    check_decode(pkg, cuda, lengths, 8, 2, 64, page, io, kept, listed=listed)


def test_decode_listed_pages_and_window(pkg, cuda):
    check_decode(pkg, cuda, [400, 90], 8, 2, 128, 32, "fp16", "fp16", window=130,
                 listed=[[[0, 1, 8, 9, 12], [11, 12]], [[0, 1, 2], [2]]])


def test_decode_extreme_scores(pkg, cuda):
    """Scores far apart in both directions: the running maximum jumps and most weights vanish."""
    lengths, hq, hk, d, page = [700, 65], 8, 2, 64, 16
    w = World(lengths, hk, d, page, "fp16")
    for b, n in enumerate(lengths):
        for t in range(n):
            w.keys[w.table[b][t // page], :, t % page] *= 0.01 if t % 97 else 20 * (1 if t % 2 else -1)
    layer, *_ = make(pkg, cuda, w, hq, hk, d, "fp16")
    q = w.normal(2, hq, d, dtype=torch.float16)
    out = layer.decode(q.view(2, -1).to(cuda), ints([n - 1 for n in lengths], cuda), w.device_table(cuda))
    for i, n in enumerate(lengths):
        exp, tol = ref.attend(q[i], w.keys, w.values, w.table[i], n - 1, page, d ** -0.5)
        close(out[i], exp, tol)


def test_decode_reports_pages_outside_the_pool(pkg, cuda):
    """Their tokens are left out, the other sequences are untouched and the next call is clean."""
    lengths, hq, hk, d, page = [100, 100, 40], 8, 2, 64, 16
    for shape in ((64, 16), (64, 8), (128, 64)):
        d, page = shape
        w = World(lengths, hk, d, page, "fp16")
        layer, *_ = make(pkg, cuda, w, hq, hk, d, "fp16")
        q = w.normal(3, hq, d, dtype=torch.float16)
        bad = [list(r) for r in w.table]
        bad[0][1], bad[2][0] = -1, 1 << 30
        pos = ints([n - 1 for n in lengths], cuda)
        out = layer.decode(q.view(3, -1).to(cuda), pos, ints(bad, cuda))
        assert layer.context.error() == -18
        for i, n in enumerate(lengths):
            exp, tol = ref.attend(q[i], w.keys, w.values, bad[i], n - 1, page, d ** -0.5)
            close(out[i], exp, tol)
        layer.decode(q.view(3, -1).to(cuda), pos, w.device_table(cuda))
        assert layer.context.error() == 0


def test_decode_reports_positions_past_the_capacity(pkg, cuda):
    w = World([50, 50], 2, 64, 16, "fp16", extra_width=0)
    layer, *_ = make(pkg, cuda, w, 8, 2, 64, "fp16")
    q = w.normal(2, 8, 64, dtype=torch.float16)
    out = layer.decode(q.view(2, -1).to(cuda), ints([64, 49], cuda), w.device_table(cuda))
    assert layer.context.error() == -12
    assert not out[0].any()
    exp, tol = ref.attend(q[1], w.keys, w.values, w.table[1], 49, 16, 0.125)
    close(out[1], exp, tol)


@pytest.mark.parametrize("page", [8, 16])
def test_decode_reports_lists_out_of_order(pkg, cuda, page):
    """A list ends before an entry that repeats, falls or lies past the position."""
    lengths, hq, hk, d = [6 * page, 6 * page, 6 * page], 4, 2, 64
    w = World(lengths, hk, d, page, "fp16")
    layer, *_ = make(pkg, cuda, w, hq, hk, d, "fp16")
    q = w.normal(3, hq, d, dtype=torch.float16)
    given = [[[0, 1, 1, 2], [2, 0, 3, 4]], [[5, 6, 7, 8], [0, -1, 2, 3]], [[-1, 0, 1, 2], [0, 1, 2, 3]]]
    used = [[[0, 1], [2]], [[5], [0]], [[], [0, 1, 2, 3]]]
    out = layer.decode(q.view(3, -1).to(cuda), ints([n - 1 for n in lengths], cuda), w.device_table(cuda),
                       pages=ints(given, cuda))
    assert layer.context.error() == -18
    for i, n in enumerate(lengths):
        exp, tol = ref.attend(q[i], w.keys, w.values, w.table[i], n - 1, page, 0.125, listed=used[i])
        close(out[i], exp, tol)


def test_decode_shared_pages(pkg, cuda):
    """Two sequences whose tables begin with the same pages."""
    w = World([100, 70], 2, 64, 16, "fp16")
    w.table[1][:3] = w.table[0][:3]
    layer, *_ = make(pkg, cuda, w, 8, 2, 64, "fp16")
    q = w.normal(2, 8, 64, dtype=torch.float16)
    out = layer.decode(q.view(2, -1).to(cuda), ints([99, 69], cuda), w.device_table(cuda))
    for i, n in enumerate([100, 70]):
        exp, tol = ref.attend(q[i], w.keys, w.values, w.table[i], n - 1, 16, 0.125)
        close(out[i], exp, tol)


@pytest.mark.parametrize("pad", [8, 3])
def test_decode_strided_pools(pkg, cuda, pad):
    """Keys and values side by side in one allocation with padded rows; 3 elements of padding break every
    16-byte alignment."""
    lengths, hq, hk, d, page = [1, 40, 77], 8, 2, 64, 16
    w = World(lengths, hk, d, page, "fp16")
    both = torch.full((2, w.keys.shape[0], page, hk, d + pad), float("nan"), dtype=torch.float16, device=cuda)
    k, v = both[0, ..., :d], both[1, ..., :d]
    k.copy_(w.keys.transpose(1, 2))
    v.copy_(w.values.transpose(1, 2))
    layer = pkg.PagedAttention(hq * d, hq, 256, k, v, {"headDim": d, "kvHeadCount": hk, "pageLayout": "NHD"})
    q = w.normal(3, hq, d, dtype=torch.float16)
    out = layer.decode(q.view(3, -1).to(cuda), ints([n - 1 for n in lengths], cuda), w.device_table(cuda))
    assert layer.context.error() == 0
    for i, n in enumerate(lengths):
        exp, tol = ref.attend(q[i], w.keys, w.values, w.table[i], n - 1, page, d ** -0.5)
        close(out[i], exp, tol)


@pytest.mark.parametrize("page", [8, 64])
def test_decode_far_pages(pkg, cuda, page):
    """Elements past 2^31 (and bytes past 2^32) from the pool's start."""
    hq, hk, d = 4, 2, 128
    row = page * hk * d
    pages = (1 << 31) // row + 70
    k, v = (torch.empty(pages, hk, page, d, dtype=torch.float16, device=cuda) for _ in range(2))
    g = torch.Generator().manual_seed(0)
    n = 2 * page + 3
    where = [pages - 1, 2, pages - 3]
    kh, vh = (torch.randn(3, hk, page, d, generator=g).half() for _ in range(2))
    for i, p in enumerate(where):
        k[p], v[p] = kh[i].to(cuda), vh[i].to(cuda)
    layer = pkg.PagedAttention(hq * d, hq, 4096, k, v, {"headDim": d, "kvHeadCount": hk})
    q = torch.randn(1, hq, d, generator=g).half()
    table = ints([where], cuda)
    out = layer.decode(q.view(1, -1).to(cuda), ints([n - 1], cuda), table)
    exp, tol = ref.attend(q[0], kh, vh, [0, 1, 2], n - 1, page, d ** -0.5)
    close(out[0], exp, tol)
    qkv = torch.randn(1, (hq + 2 * hk) * d, generator=g).half()
    layer.append(qkv.to(cuda), ints([n], cuda), table)
    assert layer.context.error() == 0
    assert torch.equal(v[where[2], :, 3].cpu(), qkv.view(-1, d)[hq + hk:])
    assert torch.equal(k[where[2], :, 3].cpu(), qkv.view(-1, d)[hq:hq + hk])


# ---------------------------------------------------------------- append
def check_append(pkg, cuda, hq, hk, d, page, io, kept, starts, chunks=None, layout="HND", behind=0, theta=10000.0,
                 bounds=True, **options):
    """chunks None: one token each. starts of -1: no sequence."""
    new = [1] * len(starts) if chunks is None else chunks
    w = World([max(s, 0) for s in starts], hk, d, page, kept, layout, room=max(new))
    layer, k, v, bd = make(pkg, cuda, w, hq, hk, d, io, bounds, ropeTheta=theta, **options)
    rows = sum(new) + behind
    qkv = w.normal(rows, (hq + 2 * hk) * d, dtype=TYPES[io])
    offsets = None
    if chunks is not None:
        offsets = ints([sum(new[:i]) for i in range(len(new) + 1)], cuda)
    query = torch.full((rows, hq * d), 7.0, dtype=TYPES[io], device=cuda)
    layer.append(qkv.to(cuda), ints(starts, cuda), w.device_table(cuda), row_offsets=offsets, query=query)
    assert layer.context.error() == 0
    row_opts = dict(theta=theta, rotary=options.get("rotaryDim"), q_norm=options.get("qNormWeight"),
                    k_norm=options.get("kNormWeight"), offset=options.get("offsetRMSNorm", False),
                    v_norm=options.get("vNorm", False))
    got_k, got_v, got_b, got_q = by_head(k, layout).cpu(), by_head(v, layout).cpu(), bd.cpu(), query.cpu()
    exp_k, exp_v, exp_b = w.keys.clone(), w.values.clone(), w.bounds.clone()
    at = 0
    for b, n in enumerate(new):
        for i in range(n):
            if starts[b] < 0:
                assert not got_q[at].any()
                at += 1
                continue
            pos = starts[b] + i
            q, kk, vv = ref.form_row(qkv[at], pos, hq, hk, d, **row_opts)
            close(got_q[at], q, ref.row_error(q, TYPES[io], d), f"query of sequence {b}, token {i}")
            p, slot = w.table[b][pos // page], pos % page
            close(got_k[p, :, slot], kk, ref.row_error(kk, w.kept, d), f"key of sequence {b}, token {i}")
            close(got_v[p, :, slot], vv, ref.row_error(vv, w.kept, d), f"value of sequence {b}, token {i}")
            exp_k[p, :, slot], exp_v[p, :, slot] = got_k[p, :, slot], got_v[p, :, slot]
            stored = got_k[p, :, slot]
            exp_b[p, :, 0] = stored if slot == 0 else torch.minimum(exp_b[p, :, 0], stored)
            exp_b[p, :, 1] = stored if slot == 0 else torch.maximum(exp_b[p, :, 1], stored)
            at += 1
    assert (got_q[at:] == 7).all()  # rows behind the last sequence
    # what no row went to is as it was (bits, NaN among them), and the bounds are those of the keys as stored
    bits = torch.int32 if w.kept == torch.float32 else torch.int16
    assert torch.equal(got_k.contiguous().view(bits), exp_k.view(bits))
    assert torch.equal(got_v.contiguous().view(bits), exp_v.view(bits))
    if bounds:
        assert torch.equal(got_b.nan_to_num(nan=99.0), exp_b.nan_to_num(nan=99.0))


APPEND_SHAPES = [(8, 2, 64), (14, 2, 64), (32, 8, 128), (16, 1, 128), (5, 5, 64)]


@pytest.mark.parametrize("io,kept", PAIRS)
@pytest.mark.parametrize("hq,hk,d", APPEND_SHAPES)
def test_append_one_token_each(pkg, cuda, hq, hk, d, io, kept):
    check_append(pkg, cuda, hq, hk, d, 16, io, kept, [0, 1, 15, 16, 31, 200, -1, 77])


@pytest.mark.parametrize("io,kept", PAIRS)
@pytest.mark.parametrize("hq,hk,d", APPEND_SHAPES)
def test_append_ragged_chunks(pkg, cuda, hq, hk, d, io, kept):
    """From the start and from inside a page, ending in one, one token, none, and rows behind the last."""
    check_append(pkg, cuda, hq, hk, d, 16, io, kept, [0, 5, 16, 30, 40, -1, 7], [50, 11, 16, 1, 0, 3, 100], behind=5)


@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("page", [1, 8, 32, 64, 512])
@pytest.mark.parametrize("chunks", [None, [70, 3, 129]])
def test_append_page_sizes_and_layouts(pkg, cuda, layout, page, chunks):
    check_append(pkg, cuda, 8, 2, 64, page, "fp16", "fp16", [0, 9, 63], chunks, layout)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("chunks", [None, [40, 1, 33]])
@pytest.mark.parametrize("io,kept", [("fp16", "fp16"), ("bf16", "bf16"), ("fp32", "fp16")])
@pytest.mark.parametrize("options", [
    {"rotaryDim": 32}, {"rotaryDim": 16}, {"rotaryDim": 24}, {"rotaryDim": 2}, {"rotaryDim": 0}, {"theta": 0.0},
    {"norms": True}, {"norms": True, "offsetRMSNorm": True, "vNorm": True}, {"vNorm": True, "bounds": False},
], ids=str)
def test_append_rotations_and_norms(pkg, cuda, d, chunks, io, kept, options):
    o = dict(options)
    if o.pop("norms", False):
        g = torch.Generator().manual_seed(1)
        o["qNormWeight"], o["kNormWeight"] = (torch.randn(d, generator=g).mul(0.3).add(1).numpy() for _ in range(2))
    check_append(pkg, cuda, 6, 2, d, 16, io, kept, [0, 17, 50], chunks, **o)


@pytest.mark.parametrize("d", [2, 8, 80, 256])
@pytest.mark.parametrize("chunks", [None, [20, 5]])
def test_append_other_head_dims(pkg, cuda, d, chunks):
    check_append(pkg, cuda, 4, 2, d, 8, "fp16", "fp16", [3, 12], chunks)
    check_append(pkg, cuda, 4, 2, d, 8, "fp32", "fp32", [3, 12], chunks)


@pytest.mark.parametrize("d", [8, 24, 72, 80, 100, 136, 200, 256])
@pytest.mark.parametrize("chunks", [None, [70, 5]])
def test_append_head_dims_normed(pkg, cuda, d, chunks):
    g = torch.Generator().manual_seed(1)
    norms = {k: torch.randn(d, generator=g).mul(0.3).add(1).numpy() for k in ("qNormWeight", "kNormWeight")}
    check_append(pkg, cuda, 4, 2, d, 32, "bf16", "bf16", [3, 12], chunks, vNorm=True, **norms)
    check_append(pkg, cuda, 13, 13, d, 64, "fp32", "fp32", [3, 12], chunks, "NHD", **norms)
    if d >= 24:
        check_append(pkg, cuda, 4, 2, d, 16, "fp32", "fp16", [3, 12], chunks, rotaryDim=16, offsetRMSNorm=True, **norms)


@pytest.mark.parametrize("io,kept", PAIRS)
def test_select_256_wide(pkg, cuda, io, kept):
    w = World([1, 640, 333, 0, 1500], 2, 256, 16, kept)
    check_select(pkg, cuda, w, 8, 2, 256, io, 9)


def test_append_far_positions(pkg, cuda):
    """Angles of far positions are reduced in 64 bits."""
    hq, hk, d, page = 4, 2, 128, 16
    k, v = (torch.zeros(2, hk, page, d, device=cuda) for _ in range(2))
    pos = [1 << 20, (1 << 24) + 5]
    width = (pos[1] // page) + 1
    table = torch.full((2, width), -1, dtype=torch.int32, device=cuda)
    table[0, pos[0] // page], table[1, pos[1] // page] = 0, 1
    layer = pkg.PagedAttention(hq * d, hq, 1 << 25, k, v, {"headDim": d, "kvHeadCount": hk, "ropeTheta": 1e6})
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(2, (hq + 2 * hk) * d, generator=g)
    query = layer.append(qkv.to(cuda), ints(pos, cuda), table)
    assert layer.context.error() == 0
    for b in range(2):
        q, kk, _ = ref.form_row(qkv[b], pos[b], hq, hk, d, theta=1e6)
        close(query[b], q, ref.row_error(q, torch.float32, d))
        close(k[b, :, pos[b] % page], kk, ref.row_error(kk, torch.float32, d))


@pytest.mark.parametrize("chunks", [None, [1, 20, 1]])
def test_append_reports_bad_pages_and_positions(pkg, cuda, chunks):
    """What has no page or no room is left out; all else is stored."""
    hq, hk, d, page = 8, 2, 64, 16
    w = World([30, 20, 63], hk, d, page, "fp16", extra_width=0)  # 64 slots per sequence at most
    layer, k, v, bd = make(pkg, cuda, w, hq, hk, d, "fp16")
    table = [list(r) for r in w.table]
    table[0][1] = w.keys.shape[0]
    rows = 3 if chunks is None else sum(chunks)
    qkv = w.normal(rows, (hq + 2 * hk) * d, dtype=torch.float16)
    offsets = None if chunks is None else ints([0, 1, 21, 22], cuda)
    query = layer.append(qkv.to(cuda), ints([30, 20, 64], cuda), ints(table, cuda), row_offsets=offsets)
    assert layer.context.error() in (-18, -12)
    assert query[:-1].any(1).all() and not query[-1].any()
    kc = k.cpu()
    x = qkv.view(rows, hq + 2 * hk, d)
    for i in range(1 if chunks is None else 12):  # from slot 20 to the end of the sequence's second page
        assert torch.equal(kc[table[1][1], :, 4 + i], x[1 + i, hq:hq + hk])
    kc[table[1][1], :, 4:] = w.keys[table[1][1], :, 4:]
    assert torch.equal(kc.view(torch.int16), w.keys.view(torch.int16))


def test_append_refuses_offsets_that_do_not_ascend_safely(pkg, cuda):
    """Offsets out of order move rows or lose them, but nothing outside the pool, the query and the table is touched."""
    w = World([0, 0, 0], 2, 64, 16, "fp16", room=32)
    layer, k, v, bd = make(pkg, cuda, w, 4, 2, 64, "fp16")
    qkv = w.normal(20, 8 * 64, dtype=torch.float16).to(cuda)
    for offsets in ([0, 30, 5, 20], [5, 3, 1, 0], [0, 0, 0, 1 << 30], [-(1 << 31), 4, 9, 20], [-5, -3, 2, 18]):
        query = layer.append(qkv, ints([0, 0, 0], cuda), w.device_table(cuda), row_offsets=ints(offsets, cuda))
        layer.context.error()
        assert query.shape == (20, 256)


# ---------------------------------------------------------------- select
def check_select(pkg, cuda, w, hq, hk, d, io, count, first=1, last=1, window=0, q=None, positions=None):
    layer, *_ = make(pkg, cuda, w, hq, hk, d, io, slidingWindow=window)
    b = len(w.lengths)
    q = w.normal(b, hq, d, dtype=TYPES[io]) if q is None else q
    positions = [n - 1 for n in w.lengths] if positions is None else positions
    got = layer.select(q.view(b, -1).to(cuda), ints(positions, cuda), w.device_table(cuda), count, first, last)
    assert layer.context.error() == 0
    exp = [ref.select(q[i], w.bounds, w.table[i], positions[i], w.page, count, first, last, window) for i in range(b)]
    assert got.tolist() == exp
    return layer, q, got


@pytest.mark.parametrize("io,kept", PAIRS)
@pytest.mark.parametrize("hq,hk,d", [(8, 2, 64), (14, 2, 64), (32, 8, 128), (16, 1, 128), (4, 4, 80)])
def test_select_matches(pkg, cuda, hq, hk, d, io, kept):
    w = World([1, 16, 17, 333, 0, 1500, 640], hk, d, 16, kept)
    check_select(pkg, cuda, w, hq, hk, d, io, 12)


@pytest.mark.parametrize("count,first,last", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (2, 1, 1), (7, 3, 4), (33, 0, 2),
                                              (94, 1, 1), (95, 1, 1), (200, 5, 5)])
def test_select_counts(pkg, cuda, count, first, last):
    w = World([1505, 40, 512], 2, 64, 16, "fp16")
    check_select(pkg, cuda, w, 8, 2, 64, "fp16", count, first, last)


@pytest.mark.parametrize("window", [1, 33, 300])
def test_select_window(pkg, cuda, window):
    w = World([1505, 40, 512], 2, 64, 16, "fp16")
    check_select(pkg, cuda, w, 8, 2, 64, "fp16", 5, window=window)


def test_select_ties_go_to_the_lower_page(pkg, cuda):
    """Many equal scores, zeros of both signs among them."""
    w = World([1280, 1280, 1280], 2, 64, 16, "fp16")
    g = torch.Generator().manual_seed(2)
    for p in range(w.bounds.shape[0]):
        w.bounds[p] = torch.randint(-1, 2, (1,), generator=g).half()
    q = torch.zeros(3, 8, 64, dtype=torch.float16)
    q[0, :, 0], q[1, :, 0] = 1, -1
    q[2] = -0.0
    check_select(pkg, cuda, w, 8, 2, 64, "fp16", 20, q=q)
    check_select(pkg, cuda, w, 8, 2, 64, "fp16", 20, 0, 0, q=q)


def test_select_many_pages(pkg, cuda):
    """More pages than one block scores, in long and short sequences."""
    w = World([20000, 16, 9000], 1, 64, 8, "fp16")
    check_select(pkg, cuda, w, 4, 1, 64, "fp16", 100)


@pytest.mark.parametrize("io,kept", PAIRS)
@pytest.mark.parametrize("d", [64, 80, 128])
def test_select_from_more_pages_than_shared_memory_ranks(pkg, cuda, io, kept, d):
    """Tables so wide that the ranks go through the workspace."""
    w = World([20000, 0, 16, 9000, 640], 1, d, 8 if d == 64 else 16, kept, extra_width=60000)
    check_select(pkg, cuda, w, 4, 1, d, io, 100)
    check_select(pkg, cuda, w, 4, 1, d, io, 7, 2, 3, window=5000)


@pytest.mark.parametrize("n", [5, 65, 200, 257, 300, 1024, 1025, 1500, 4000])
@pytest.mark.parametrize("batch", [1, 3, 40])
def test_select_block_and_cluster_sizes(pkg, cuda, n, batch):
    """Around the sizes where the blocks and the clusters change."""
    batch = min(batch, 6000 // n)  # (the 64-bit form on the host is slow)
    w = World([max(1, n * 8 - 3 * i) for i in range(batch)], 2, 64, 8, "fp16")
    check_select(pkg, cuda, w, 8, 2, 64, "fp16", max(2, n // 5))


@pytest.mark.parametrize("wide", [1, 300, 1200, 2000])
@pytest.mark.parametrize("batch", [30, 74, 90, 200])
def test_select_many_sequences(pkg, cuda, wide, batch):
    """Blocks and clusters by the number of sequences, few of them as long as the table."""
    w = World([(900, 8, 70, 0, 1)[i % 5] + i % 3 for i in range(batch)], 2, 64, 8, "bf16", extra_width=wide)
    check_select(pkg, cuda, w, 4, 2, 64, "bf16", 7)


def test_select_tiny_and_huge_keys(pkg, cuda):
    """Subnormal bounds and the type's largest values."""
    for kept, tiny in (("fp16", 2.0 ** -24), ("bf16", 2.0 ** -130)):
        w = World([640, 640], 2, 64, 16, kept)
        w.bounds.mul_(tiny * 8) if kept == "fp16" else w.bounds.mul_(tiny)
        check_select(pkg, cuda, w, 8, 2, 64, kept, 9)
        w.bounds.copy_(torch.randn(w.bounds.shape, generator=w.g).sign() * torch.finfo(w.kept).max
                       * torch.rand(w.bounds.shape, generator=w.g).clamp(min=0.25))
        check_select(pkg, cuda, w, 8, 2, 64, kept, 9, q=w.normal(2, 8, 64, dtype=w.kept) * 1e-3)


def test_select_reports_pages_outside_the_pool(pkg, cuda):
    w = World([320, 64], 2, 64, 16, "fp16")
    w.table[0][3] = 1 << 20
    layer, *_ = make(pkg, cuda, w, 8, 2, 64, "fp16")
    q = w.normal(2, 8, 64, dtype=torch.float16)
    got = layer.select(q.view(2, -1).to(cuda), ints([319, 63], cuda), w.device_table(cuda), 6)
    assert layer.context.error() == -18
    assert got.tolist() == [ref.select(q[i], w.bounds, w.table[i], n - 1, 16, 6) for i, n in enumerate([320, 64])]


# ---------------------------------------------------------------- refusals
def test_python_refuses(pkg, cuda):
    k, v = (torch.zeros(4, 2, 16, 64, dtype=torch.float16, device=cuda) for _ in range(2))
    bounds = torch.zeros(4, 2, 2, 64, dtype=torch.float16, device=cuda)

    def layer(key=k, value=v, options=None, key_bounds=bounds, heads=8):
        o = {"headDim": 64, "kvHeadCount": 2, "maxBatch": 4, **(options or {})}
        return pkg.PagedAttention(heads * 64, heads, 64, key, value, o, key_bounds=key_bounds)

    for kw, err in [(dict(key=k.double()), TypeError), (dict(value=v.float()), TypeError), (dict(key=k.cpu()), TypeError),
                    (dict(key=k[:, :1]), ValueError), (dict(value=v.transpose(1, 2).contiguous().transpose(1, 2)), ValueError),
                    (dict(key=k.transpose(2, 3), value=v.transpose(2, 3)), ValueError),
                    (dict(options={"pageLayout": "NHD"}), ValueError), (dict(options={"pageLayout": "x"}), ValueError),
                    (dict(options={"dtype": torch.float64}), TypeError), (dict(key_bounds=bounds.float()), TypeError),
                    (dict(key_bounds=bounds[:2]), ValueError), (dict(options={"qNormWeight": [1.0] * 3}), ValueError),
                    (dict(value=k), pkg.TlaError), (dict(options={"dtype": torch.bfloat16}), pkg.TlaError),
                    (dict(heads=9), pkg.TlaError), (dict(key=k.expand(4, 2, 16, 64)[:, :, ::3], value=v[:, :, ::3]), pkg.TlaError)]:
        with pytest.raises(err):
            layer(**kw)
    a = layer()
    q = torch.zeros(2, 512, dtype=torch.float16, device=cuda)
    qkv = torch.zeros(2, 768, dtype=torch.float16, device=cuda)
    pos, table = ints([0, 0], cuda), ints([[0], [1]], cuda)
    a.decode(q, pos, table)
    a.append(qkv, pos, table)
    bad = [
        (lambda: a.decode(q.float(), pos, table), TypeError), (lambda: a.decode(q.cpu(), pos, table), TypeError),
        (lambda: a.decode(q[:, ::2], pos, table), TypeError), (lambda: a.decode(q[:1], pos, table), ValueError),
        (lambda: a.decode(q, pos.long(), table), TypeError), (lambda: a.decode(q, pos, table[:1]), ValueError),
        (lambda: a.decode(q, pos, table.long()), TypeError), (lambda: a.decode(q, pos[:, None], table), ValueError),
        (lambda: a.decode(q, pos, table[:, :0]), pkg.TlaError), (lambda: a.decode(q, pos, table, gate=q[:1]), ValueError),
        (lambda: a.decode(q, pos, table, out=q.float()), TypeError),
        (lambda: a.decode(q, pos, table, pages=ints([[[0]], [[0]]], cuda)), ValueError),
        (lambda: a.decode(q, pos, table, pages=torch.zeros(2, 2, 0, dtype=torch.int32, device=cuda)), pkg.TlaError),
        (lambda: a.append(qkv[:1], pos, table), ValueError), (lambda: a.append(q, pos, table), ValueError),
        (lambda: a.append(qkv, pos, table, row_offsets=pos), ValueError),
        (lambda: a.append(qkv, pos, table, query=qkv), ValueError),
        (lambda: a.select(q, pos, table, 0), pkg.TlaError), (lambda: a.select(q, pos, table, 2, 2, 1), pkg.TlaError),
        (lambda: a.select(q, pos, table, 2, -1, 1), pkg.TlaError), (lambda: a.select(q, pos, table, -3), pkg.TlaError),
        (lambda: layer(key_bounds=None).select(q, pos, table, 2), pkg.TlaError),
        (lambda: layer(options={"attnScale": -1.0}).select(q, pos, table, 2), pkg.TlaError),
        (lambda: layer(options={"maxBatch": 1}).decode(q, pos, table), pkg.TlaError),
        (lambda: a.decode(q, pos, table, out=q), pkg.TlaError),                              # outputs over inputs
        (lambda: a.append(qkv, pos, table, query=qkv.view(-1)[512:1536].view(2, 512)), pkg.TlaError),
    ]
    for call, err in bad:
        with pytest.raises(err):
            call()
    a.close()
    with pytest.raises(pkg.TlaError):
        a.decode(q, pos, table)
    # a long table's call needs a workspace, and refuses none or a small one
    long = pkg.PagedAttention(512, 8, 1 << 16, k, v, {"headDim": 64, "kvHeadCount": 2})
    wide = torch.zeros(2, 4096, dtype=torch.int32, device=cuda)
    need = ctypes.c_size_t()
    assert pkg.lib().tla_paged_workspace(long.handle, 2, 4096, 0, ctypes.byref(need), None) == 0 and need.value > 0
    work = torch.empty(need.value + 16, dtype=torch.uint8, device=cuda)
    for at, size in ((None, 0), (work.data_ptr(), need.value - 1), (work.data_ptr() + 8, need.value)):
        assert pkg.lib().tla_paged_decode(long.handle, q.data_ptr(), pos.data_ptr(), wide.data_ptr(), 4096, None, 0,
                                          None, q.data_ptr(), 2, at, size, None) == -1


def test_overlaps_and_short_workspaces_are_refused(pkg, cuda):
    k, v = (torch.zeros(4, 2, 16, 64, dtype=torch.float16, device=cuda) for _ in range(2))
    bounds = torch.zeros(4, 2, 2, 64, dtype=torch.float16, device=cuda)
    a = pkg.PagedAttention(512, 8, 1 << 16, k, v, {"headDim": 64, "kvHeadCount": 2}, key_bounds=bounds)
    lib, pos, table = pkg.lib(), ints([3, 3], cuda), torch.zeros(2, 4096, dtype=torch.int32, device=cuda)
    buf = torch.zeros(2 * 768 + 4096, dtype=torch.float16, device=cuda)
    at, end = buf.data_ptr(), buf.data_ptr() + 2 * 768 * 2
    need, choose = ctypes.c_size_t(), ctypes.c_size_t()
    assert lib.tla_paged_workspace(a.handle, 2, 4096, 0, ctypes.byref(need), ctypes.byref(choose)) == 0 and need.value
    work = torch.empty(need.value + choose.value + 16, dtype=torch.uint8, device=cuda)

    def decode(out, w=work.data_ptr(), size=need.value, gate=None):
        return lib.tla_paged_decode(a.handle, at, pos.data_ptr(), table.data_ptr(), 4096, None, 0, gate, out, 2, w, size,
                                    None)

    def select(out):
        return lib.tla_paged_select(a.handle, at, pos.data_ptr(), table.data_ptr(), 4096, 1, 1, out, 4, 2,
                                    work.data_ptr(), choose.value, None)

    assert decode(end) == 0 and decode(end, gate=end) == 0 and select(end) == 0
    assert decode(end, None, 0) == decode(end, size=need.value - 1) == decode(end, work.data_ptr() + 8) == -1
    assert decode(at) == decode(at + 2 * 512 * 2 - 16) == decode(end, gate=end + 16) == -1
    assert select(at) == select(at + 2 * 512 * 2 - 16) == -1
    for out in (at, end - 16):
        assert lib.tla_paged_append(a.handle, at, pos.data_ptr(), None, table.data_ptr(), 4096, 2, 2, out, None) == -1
    torch.cuda.synchronize()


def test_append_refuses_rows_that_do_not_fit(pkg, cuda):
    """A head_dim that goes through shared memory row by row, with more heads than it holds."""
    k, v = (torch.zeros(2, 64, 4, 84, dtype=torch.float16, device=cuda) for _ in range(2))
    a = pkg.PagedAttention(640 * 84, 640, 8, k, v, {"headDim": 84, "kvHeadCount": 64})
    with pytest.raises(pkg.TlaError, match="UNSUPPORTED"):
        a.append(torch.zeros(1, 768 * 84, dtype=torch.float16, device=cuda), ints([0], cuda), ints([[0]], cuda))
    torch.zeros(1, device=cuda)  # no CUDA error is left behind


def test_append_many_heads(pkg, cuda):
    check_append(pkg, cuda, 640, 64, 80, 4, "fp16", "fp16", [0, 5])


def test_decode_gate_as_output(pkg, cuda):
    w = World([70, 40], 2, 64, 16, "fp16")
    layer, *_ = make(pkg, cuda, w, 8, 2, 64, "fp16")
    q, gate = (w.normal(2, 512, dtype=torch.float16).to(cuda) for _ in range(2))
    pos, table = ints([69, 39], cuda), w.device_table(cuda)
    exp = layer.decode(q, pos, table, gate=gate)
    assert torch.equal(layer.decode(q, pos, table, gate=gate, out=gate), exp)


def test_empty_calls(pkg, cuda):
    k, v = (torch.zeros(4, 2, 16, 64, dtype=torch.float16, device=cuda) for _ in range(2))
    a = pkg.PagedAttention(512, 8, 64, k, v, {"headDim": 64, "kvHeadCount": 2})
    none, table = ints([], cuda), torch.zeros(0, 3, dtype=torch.int32, device=cuda)
    assert a.decode(torch.zeros(0, 512, dtype=torch.float16, device=cuda), none, table).shape == (0, 512)
    assert a.append(torch.zeros(0, 768, dtype=torch.float16, device=cuda), none, table).shape == (0, 512)
    assert a.append(torch.zeros(0, 768, dtype=torch.float16, device=cuda), ints([5], cuda), ints([[0]], cuda),
                    row_offsets=ints([0, 0], cuda)).shape == (0, 512)


# ---------------------------------------------------------------- the operators together
OPTIONS = {"headDim": 64, "kvHeadCount": 2, "ropeTheta": 10000.0}


def test_prompts_then_steps_match_the_contiguous_layer(pkg, cuda):
    """Prompts of different lengths, then decode steps with pages handed out as the sequences grow: the
    same outputs as CUDAAttention over its contiguous cache, within both paths' fp16 roundings, dense and
    with every page selected."""
    hq, hk, d, page, room = 8, 2, 64, 16, 96
    prompts, steps = [37, 5, 64], 20
    g = torch.Generator().manual_seed(5)
    dense = pkg.CUDAAttention(None, hq * d, hq, room, {**OPTIONS, "maxBatch": 3, "dtype": torch.float16})
    pages = 3 * room // page
    k, v = (torch.full((pages, hk, page, d), float("nan"), dtype=torch.float16, device=cuda) for _ in range(2))
    bounds = torch.full((pages, hk, 2, d), float("nan"), dtype=torch.float16, device=cuda)
    paged = pkg.PagedAttention(hq * d, hq, room, k, v, OPTIONS, key_bounds=bounds)
    free = torch.randperm(pages, generator=g).tolist()
    table = [[-1] * (room // page) for _ in prompts]

    def hold(b, n):
        for i in range(-(-n // page)):
            if table[b][i] < 0:
                table[b][i] = free.pop()

    rows = [torch.randn(n, (hq + 2 * hk) * d, generator=g).half().to(cuda) for n in prompts]
    for b, n in enumerate(prompts):
        hold(b, n)
        padded = torch.zeros(3, n, (hq + 2 * hk) * d, dtype=torch.float16, device=cuda)
        padded[b] = rows[b]
        dense.prefill(padded, ints([0, 0, 0], cuda))  # (the other rows are overwritten by their own prompt)
        for c in range(b):
            again = torch.zeros(3, prompts[c], (hq + 2 * hk) * d, dtype=torch.float16, device=cuda)
            again[c] = rows[c]
    # each sequence's prompt last: prefill the rectangle of all prompts, then steps overwrite what lies past them
    longest = max(prompts)
    block = torch.zeros(3, longest, (hq + 2 * hk) * d, dtype=torch.float16, device=cuda)
    for b, n in enumerate(prompts):
        block[b, :n] = rows[b]
    dense.prefill(block, ints([0, 0, 0], cuda))
    offsets = [0, prompts[0], prompts[0] + prompts[1], sum(prompts)]
    paged.append(torch.cat(rows), ints([0, 0, 0], cuda), ints(table, cuda), row_offsets=ints(offsets, cuda))
    for s in range(steps):
        positions = [n + s for n in prompts]
        for b, n in enumerate(positions):
            hold(b, n + 1)
        qkv = torch.randn(3, (hq + 2 * hk) * d, generator=g).half().to(cuda)
        pos, t = ints(positions, cuda), ints(table, cuda)
        exp = dense.decode(qkv, pos).float()
        q = paged.append(qkv, pos, t)
        out = paged.decode(q, pos, t)
        # both round P and the output to fp16 (2^-11 each, relative to values of at most 4 in this data)
        assert (out.float() - exp).abs().max() <= 4 * 4 * 2.0 ** -11
        every = paged.select(q, pos, t, room // page)
        assert torch.equal(every[:, 0, 0], torch.zeros(3, dtype=torch.int32, device=cuda))
        assert (paged.decode(q, pos, t, pages=every).float() - out.float()).abs().max() <= 4 * 4 * 2.0 ** -11
    assert paged.context.error() == 0
    for b, n in enumerate(prompts):
        dk, dv = dense.read_cache(b, 0, n + steps)
        at = torch.tensor([[table[b][t // page], t % page] for t in range(n + steps)], device=cuda)
        pk = k[at[:, 0], :, at[:, 1]].reshape(n + steps, -1).float().cpu()
        assert (pk - torch.from_numpy(dk)).abs().max() <= 2.0 ** -10 * 8  # one fp16 step of values under 8
        assert torch.equal(v[at[:, 0], :, at[:, 1]].reshape(n + steps, -1).float().cpu(), torch.from_numpy(dv))


def step(layer, qkv, pos, table, count):
    q = layer.append(qkv, pos, table)
    pages = layer.select(q, pos, table, count)
    return q, layer.decode(q, pos, table), pages, layer.decode(q, pos, table, pages=pages)


def serving(pkg, cuda, seed, hq=8, hk=2, d=64, lengths=(300, 17, 650), context=None, extra_width=1):
    w = World(list(lengths), hk, d, 16, "fp16", seed=seed, room=1, extra_width=extra_width)
    k, v, bd = w.device_pool(cuda)
    layer = pkg.PagedAttention(hq * d, hq, w.width * 16, k, v, {"headDim": d, "kvHeadCount": hk, "ropeTheta": 1e4},
                               key_bounds=bd, context=context)
    qkv = w.normal(len(lengths), (hq + 2 * hk) * d, dtype=torch.float16).to(cuda)
    return layer, qkv, ints(list(lengths), cuda), w.device_table(cuda)


def test_two_graphs_and_an_eager_call_at_once(pkg, cuda):
    """Steps of two layers of one context captured into two graphs, replayed on two streams at the same time
    beside eager steps of a third: each equals its own eager step, bit for bit."""
    worlds = [serving(pkg, cuda, s, lengths=n, extra_width=x)
              for s, (n, x) in enumerate([((300, 17, 650), 1), ((2000,), WIDE), ((40, 999), WIDE)])]
    exp = [[t.clone() for t in step(*w, 8)] for w in worlds]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in worlds]
    for w in worlds[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*w, 8))
        graphs.append(g)
    for t in [x for o in outs for x in o]:
        t.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = step(*worlds[2], 8)
    torch.cuda.synchronize()
    for got, e in zip(outs + [eager], exp):
        for a, b in zip(got, e):
            assert torch.equal(a, b)
    assert worlds[0][0].context.error() == 0


def test_graph_follows_positions_and_tables(pkg, cuda):
    """A captured step replayed with other positions, pages and rows: what the buffers hold at the replay counts."""
    layer, qkv, pos, table = serving(pkg, cuda, 3)
    step(layer, qkv, pos, table, 4)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step(layer, qkv, pos, table, 4)
    pos.copy_(ints([5, -1, 200], cuda))
    table.copy_(table.roll(1, 1))
    table[:, 0] = table[:, -1].clamp(min=0)
    table.clamp_(min=0)
    qkv.mul_(-0.5)
    layer.valuePages.nan_to_num_(nan=0.0)
    layer.keyPages.nan_to_num_(nan=0.0)
    layer.keyBounds.nan_to_num_(nan=0.0)
    g.replay()
    got = [t.clone() for t in outs]
    exp = step(layer, qkv, pos, table, 4)
    for a, b in zip(got, exp):
        assert torch.equal(a, b)
    assert not got[1][1].any() and (got[2][1] == -1).all()


def test_given_stream(pkg, cuda):
    """A call on a stream that is not the current one runs there: behind that stream's earlier work."""
    layer, qkv, pos, table = serving(pkg, cuda, 4)
    exp = step(layer, qkv, pos, table, 6)
    s = torch.cuda.Stream()
    held = qkv.clone()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        qkv.zero_()
        torch.cuda._sleep(20_000_000)
        qkv.copy_(held)
    q = layer.append(qkv, pos, table, stream=s)
    pages = layer.select(q, pos, table, 6, stream=s)
    out = layer.decode(q, pos, table, pages=pages, stream=s)
    s.synchronize()
    assert torch.equal(q, exp[0]) and torch.equal(pages, exp[2]) and torch.equal(out, exp[3])


@pytest.mark.parametrize("wide", [1, WIDE])
def test_repeated_calls_agree_bit_for_bit(pkg, cuda, wide):
    layer, qkv, pos, table = serving(pkg, cuda, 6, 32, 8, 128, (4000, 3, 777, 0, 129), extra_width=wide)
    first = [t.clone() for t in step(layer, qkv, pos, table, 16)]
    for _ in range(10):
        for a, b in zip(step(layer, qkv, pos, table, 16), first):
            assert torch.equal(a, b)


def test_paged_under_bounds_check_build(pkg):
    """Most of these tests in a fresh process that loads libtla_check.so: no guarded index may leave its buffer."""
    if os.environ.get("TLA_LIBRARY"):
        pytest.skip("runs in that process")
    root = Path(__file__).resolve().parent.parent
    subprocess.run(["make", "-s", "-j8", "-C", str(root / "three-llm_b200" / "csrc"), "check"], check=True)
    env = dict(os.environ, TLA_LIBRARY=str(root / "three-llm_b200" / "libtla_check.so"))
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-p", "no:cacheprovider", "-m", "gpu",
                        "tests/test_paged_gpu.py", "-k",
                        "not in_shares_shapes and not block_and_cluster and not more_pages"], cwd=root, env=env, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-2000:]
    assert " passed" in r.stdout
