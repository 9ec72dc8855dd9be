"""Edges of the paged cache on the GPU, at sizes and values where a rounding, a
limit or an address goes wrong. Worlds and 64-bit forms are those of
test_paged_gpu.py and paged_ref.py."""
import math
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from oracle import oracle
from tests import paged_ref as ref
from tests.test_paged_gpu import PAIRS, TYPES, WIDE, World, by_head, close, ints, make

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent


@pytest.mark.parametrize("page", [8, 16])
@pytest.mark.parametrize("wide", [1, WIDE])
def test_decode_reports_what_follows_a_full_list(pkg, cuda, page, wide):
    """A list that names every page of the sequence and goes on with something else than a negative entry."""
    w = World([3 * page - 2, 3 * page - 2], 1, 64, page, "fp16", extra_width=wide)
    layer, *_ = make(pkg, cuda, w, 4, 1, 64, "fp16")
    q, pos, table = w.normal(2, 256, dtype=torch.float16).to(cuda), ints([3 * page - 3] * 2, cuda), w.device_table(cuda)
    exp = layer.decode(q, pos, table)
    assert layer.context.error() == 0
    for tail, code in ((-1, 0), (3, -18), (0, -18), (1 << 30, -18)):
        out = layer.decode(q, pos, table, pages=ints([[[0, 1, 2, -1]], [[0, 1, 2, tail]]], cuda))
        assert layer.context.error() == code
        # (the same tokens, perhaps in other shares: both round weights and output once)
        assert (out.float() - exp.float()).abs().max() <= 4 * 2.0 ** -10


@pytest.mark.parametrize("d,io,kept", [(64, "fp16", "fp16"), (128, "bf16", "bf16"), (96, "fp32", "fp16"), (256, "fp32", "fp32"),
                                       (100, "fp16", "fp16"), (100, "fp32", "fp32"), (64, "fp32", "bf16")])
@pytest.mark.parametrize("chunks", [[1, 1, 1], [40, 1, 33], None])
def test_append_bounds_leave_out_what_is_no_number(pkg, cuda, d, io, kept, chunks):
    """NaN keys are stored but not counted, first and last slots among them, however the tokens were appended."""
    hk, page, n = 2, 16, 48
    w = World([0, 0, 0], hk, d, page, kept, room=n)
    layer, k, v, bd = make(pkg, cuda, w, hk, hk, d, io, rotaryDim=0)
    x = w.normal(3, n, 3 * hk * d, dtype=TYPES[io])
    keys = x.view(3, n, 3, hk, d)[:, :, 1]
    keys[torch.rand(keys.shape, generator=w.g) < 0.3] = float("nan")
    keys[:, 0::16, :, 1] = float("nan")
    keys[:, 15::16, :, 2] = float("nan")
    keys[:, 3::16, :] = w.normal(*keys[:, 3::16].shape, dtype=TYPES[io])  # one number at least
    table = w.device_table(cuda)
    at = [0, 0, 0]
    while min(at) < n:  # to 48 tokens each, from the start
        new = [min(c, n - a) for c, a in zip(chunks or [n, n, n], at)]
        rows = torch.cat([x[b, a:a + c] for b, (a, c) in enumerate(zip(at, new))]).to(cuda)
        offsets = None
        if new != [1, 1, 1] or chunks != [1, 1, 1]:
            offsets = ints([0, new[0], new[0] + new[1], sum(new)], cuda)
        layer.append(rows, ints(at, cuda), table, row_offsets=offsets)
        at = [a + c for a, c in zip(at, new)]
        if chunks == [40, 1, 33]:
            chunks = [5, 20, 1]
    assert layer.context.error() == 0
    stored = keys.to(w.kept).float().view(3, n // page, page, hk, d)
    low, high = stored.nan_to_num(nan=float("inf")).amin(2), stored.nan_to_num(nan=float("-inf")).amax(2)
    for b in range(3):
        for i in range(n // page):
            p = w.table[b][i]
            assert torch.equal(bd[p, :, 0].float().cpu(), low[b, i]) and torch.equal(bd[p, :, 1].float().cpu(), high[b, i])


# ---------------------------------------------------------------- select: tables next to the 48 KB default
SELECT_TABLES = """
import sys
sys.path.insert(0, {root!r})
import torch
import __graft_entry__ as ge
from tests.test_paged_gpu import World, check_select
pkg, cuda = ge.load_package(), torch.device("cuda", 0)
d, batch = {d}, {batch}
for pages in (9200, 9700, 10240, 11200, 11700, 12000, 12288):  # ascending: no call is covered by a larger one before it
    w = World([900, 16, 333, 0] + [40] * (batch - 4), 2, d, 8, "fp16")
    w.table = [row[:w.width] + [-7] * (pages - w.width) for row in w.table]
    w.width = pages
    check_select(pkg, cuda, w, 4, 2, d, "fp16", 7)
print("all tables done")
"""


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("batch", [4, 80])
def test_select_from_tables_near_the_default_shared_memory(pkg, cuda, d, batch):
    """Ranks that fit 48 KB by themselves but not beside the block's own variables, each width the largest of its
    process so far; few pairs run in blocks of 512 threads, many in blocks of 256."""
    r = subprocess.run([sys.executable, "-c", SELECT_TABLES.format(root=str(ROOT), d=d, batch=batch)], cwd=ROOT,
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "all tables done" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


# ---------------------------------------------------------------- errors
def test_a_failed_call_leaves_no_error_for_the_next(pkg, cuda):
    """A refused allocation is reported by its own call and not by a later launch."""
    small = pkg.CUDAAttention(None, 160, 2, 16, {"headDim": 80, "ropeTheta": 1e4})
    qkv, pos = torch.ones(1, 480, dtype=torch.float16, device=cuda), ints([0], cuda)
    exp = small.decode(qkv, pos)
    with pytest.raises(pkg.TlaError, match="OUT_OF_MEMORY"):
        pkg.CUDAAttention(None, 64 * 256, 64, (1 << 31) - 1, {"headDim": 256, "maxBatch": 1024})
    assert torch.equal(small.decode(qkv, pos), exp)


# ---------------------------------------------------------------- decode: the weights' roundings
def places(w, n):
    """(pages, slots) of the first sequence's n tokens."""
    t = torch.arange(n)
    return torch.tensor(w.table[0])[t // w.page], t % w.page


def dominated(n, d, page, kept, gaps, wide, every):
    """One sequence, one kv head: token 5 and each `every`-th after it have the top score and values of zeros, the
    others lie `gaps` below it in powers of two (given attnScale = ln 2 and the query (1, 0, ...)), so that the output
    is what they sum up to."""
    w = World([n], 1, d, page, kept, extra_width=wide)
    p, s = places(w, n)
    below = torch.tensor(gaps, dtype=torch.float64)[torch.arange(n) % len(gaps)]
    top = torch.arange(5, n, every)
    below[top] = 0
    w.keys[p, 0, s] = 0
    w.keys[p, 0, s, 0] = (8.0 - below).to(w.kept)
    w.values[p, 0, s] = (w.values[p, 0, s].abs() + 0.5) * 4096
    w.values[p[top], 0, s[top]] = 0
    return w


def check_dominated(pkg, cuda, w, n, hq, d, io, kept):
    layer, *_ = make(pkg, cuda, w, hq, 1, d, io, attnScale=math.log(2.0))
    q = torch.zeros(1, hq, d, dtype=TYPES[io])
    q[..., 0] = 1
    out = layer.decode(q.view(1, -1).to(cuda), ints([n - 1], cuda), w.device_table(cuda))
    assert layer.context.error() == 0
    p, s = places(w, n)
    k, v = w.keys[p, 0, s].double(), w.values[p, 0, s].double()
    weight = torch.softmax(k[:, 0] * math.log(2.0), 0)
    exp = weight @ v
    # A score carries the roundings of its product, the scale and log2(e), 2^-22 of at most 32 powers of two; the sums
    # run in 32 bits over n / 16 steps spread over 32 warps at least, then 24 joins, 2^-22 each (the tensor cores cut
    # off). A weight is kept in 22 bits (two fp16 parts), 11 or 8, and its smallest part no finer than 2^-39 of the
    # largest (fp16: half of 2^-24 under a top of 2^14).
    share = 32 * 2.0 ** -22 * 2 + (n / 16 / 32 + 24) * 2.0 ** -22
    share += {"fp32": 2.0 ** -21, "fp16": 2 * 2.0 ** -11, "bf16": 2 * 2.0 ** -8}[io]
    tol = share * exp + (0 if io == "bf16" else n * 2.0 ** -39 * v.max() / (weight / weight.max()).sum())
    tol = tol + ref.half_step(TYPES[io]) * exp + ref.smallest(TYPES[io])
    for h in range(hq):
        close(out[0].view(hq, d)[h], exp, tol, f"head {h}")


@pytest.mark.parametrize("io,kept", [("fp32", "fp16"), ("fp16", "fp16"), ("bf16", "bf16"), ("fp32", "fp32")])
@pytest.mark.parametrize("gap", [12.0, 20.0, 24.40625, 25.203125, 26.0])
@pytest.mark.parametrize("d,wide", [(64, 1), (64, WIDE), (128, 1), (256, 1)])
@pytest.mark.parametrize("every", [16, 10000])
def test_decode_many_small_weights(pkg, cuda, io, kept, gap, d, wide, every):
    """Thousands of equal weights far below one, among few large ones or beside a single one: together they count, and
    equal roundings add up."""
    w = dominated(8193, d, 16, kept, [gap], wide, every)
    check_dominated(pkg, cuda, w, 8193, 8, d, io, kept)


@pytest.mark.parametrize("io,kept", [("fp32", "fp16"), ("fp16", "fp16"), ("bf16", "bf16")])
@pytest.mark.parametrize("hq", [3, 16])
def test_decode_weights_of_every_size(pkg, cuda, io, kept, hq):
    w = dominated(4097, 64, 32, kept, [1.0 + 0.25 * i for i in range(107)], 1, 16)
    check_dominated(pkg, cuda, w, 4097, hq, 64, io, kept)


@pytest.mark.parametrize("io,kept", [("fp32", "fp16"), ("fp16", "fp16"), ("bf16", "bf16"), ("fp32", "bf16"), ("fp32", "fp32")])
@pytest.mark.parametrize("top", [2.0 ** e for e in (0, 10, 20, 24, 25, 26, 27, 28, 29, 30)])
def test_decode_equal_scores_of_any_size(pkg, cuda, io, kept, top):
    """The same key everywhere, its score up to where a float's step is larger than any weight's exponent: the mean of
    the values."""
    n, d, page = 333, 64, 16
    w = World([n], 1, d, page, kept)
    p, s = places(w, n)
    w.keys[p, 0, s] = 0
    w.keys[p, 0, s, 0] = 2.0 ** 15
    layer, *_ = make(pkg, cuda, w, 4, 1, d, io, attnScale=1.0)
    q = torch.zeros(1, 4, d, dtype=TYPES[io])
    q[..., 0] = top / 2 ** 15
    out = layer.decode(q.view(1, -1).to(cuda), ints([n - 1], cuda), w.device_table(cuda))
    v = w.values[p, 0, s].double()
    size = v.abs().mean(0)
    # equal weights: what they are rounded to cancels; sums in 32 bits, then the output's own rounding
    tol = 64 * 2.0 ** -22 * size + ref.half_step(TYPES[io]) * v.mean(0).abs() + ref.smallest(TYPES[io])
    for h in range(4):
        close(out.view(4, d)[h], v.mean(0), tol)


def worst_gap(dtype, low, high):
    """The number of the type between low and high whose weight 2^-gap is furthest from the type's own, relative to it."""
    gap = torch.arange(low, high, torch.finfo(dtype).eps, dtype=torch.float64).to(dtype).double().unique()
    weight = torch.exp2(-gap)
    return float(gap[((weight.to(dtype).double() - weight).abs() / weight).argmax()])


@pytest.mark.parametrize("io,kept", [("fp32", "fp16"), ("fp16", "fp16"), ("bf16", "bf16")])
@pytest.mark.parametrize("wide", [1, WIDE])
@pytest.mark.parametrize("low", [0.5, 1.5, 4.5])
def test_decode_gives_a_constant_back(pkg, cuda, io, kept, wide, low):
    """Where all values are one number, the output is that number whatever the weights are rounded to: the sum is of
    the weights that the values are multiplied with."""
    n, d, page = 700, 64, 16
    w = World([n], 1, d, page, kept, extra_width=wide)
    p, s = places(w, n)
    c = 2 - 2 * torch.finfo(w.kept).eps  # of all numbers the one whose half step is the smallest part of it, or nearly
    w.keys[p, 0, s] = 0
    w.keys[p[5::16], 0, s[5::16], 0] = worst_gap(w.kept, low, low + 0.5)
    w.values[p, 0, s] = c
    layer, *_ = make(pkg, cuda, w, 8, 1, d, io, attnScale=math.log(2.0))
    q = torch.zeros(1, 8, d, dtype=TYPES[io])
    q[..., 0] = 1
    out = layer.decode(q.view(1, -1).to(cuda), ints([n - 1], cuda), w.device_table(cuda)).double().cpu()
    # float32: weights in two parts against their 32-bit sum, and at most 40 additions of either, 2^-23 each; the
    # 16-bit types have the constant's neighbours further off than that
    assert (out - c).abs().max() <= (2.0 ** -17 * c if io == "fp32" else 0.0)


@pytest.mark.parametrize("io,kept", [("fp32", "fp16"), ("fp16", "fp16"), ("bf16", "bf16")])
@pytest.mark.parametrize("wide", [1, WIDE])
@pytest.mark.parametrize("d,hq", [(64, 4), (64, 16), (128, 7), (256, 8)])
def test_decode_rounds_nothing_but_its_output(pkg, cuda, io, kept, wide, d, hq):
    """Two weights, one of them as far from the 16-bit type as they come, whose shares of the output nearly cancel: what
    the weights were rounded to would be most of what is left."""
    n, page = 700, 16
    w = World([n], 1, d, page, kept, extra_width=wide)
    p, s = places(w, n)
    gap = worst_gap(w.kept, 0.5, 1.0)
    w.keys[p, 0, s] = 0
    w.keys[p[::2], 0, s[::2], 0] = gap
    w.values[p[::2], 0, s[::2]] = 1
    w.values[p[1::2], 0, s[1::2]] = -2.0 ** gap
    layer, *_ = make(pkg, cuda, w, hq, 1, d, io, attnScale=math.log(2.0))
    q = torch.zeros(1, hq, d, dtype=TYPES[io])
    q[..., 0] = 1
    out = layer.decode(q.view(1, -1).to(cuda), ints([n - 1], cuda), w.device_table(cuda))
    weight = torch.softmax(w.keys[p, 0, s, 0].double() * math.log(2.0), 0)
    v = w.values[p, 0, s].double()
    exp, size = weight @ v, weight @ v.abs()
    # a score of at most one power of two, its roundings and the exponential's 2^-22; 700 / 16 steps over four warps and
    # 24 joins, 2^-22 each; a weight's two parts, 21 bits or 15
    share = 2 * 2.0 ** -22 + (700 / 16 / 4 + 24) * 2.0 ** -22 + (2.0 ** -15 if kept == "bf16" else 2.0 ** -21)
    tol = share * size + ref.half_step(TYPES[io]) * exp.abs() + ref.smallest(TYPES[io])
    for h in range(hq):
        close(out[0].view(hq, d)[h], exp, tol, f"head {h}")


FORMS = [(64, "fp16", "fp16", 16), (128, "bf16", "bf16", 16), (64, "fp32", "fp16", 32), (256, "fp32", "fp16", 16),
         (64, "fp32", "fp32", 16), (128, "fp32", "bf16", 16), (64, "bf16", "bf16", 4), (100, "fp16", "fp16", 16)]


@pytest.mark.parametrize("d,io,kept,page", FORMS)
@pytest.mark.parametrize("wide", [1, WIDE])
def test_decode_infinite_values(pkg, cuda, d, io, kept, page, wide):
    """An infinite value that takes part is one in its dimension of the output, whatever its weight is made of, and
    nowhere else."""
    n, hq, inf = 400, 6, float("inf")
    w = World([n] * 2, 2, d, page, kept, extra_width=wide)
    w.values[w.table[0][0], 0, 0, 3] = inf
    w.values[w.table[1][33 // page], 1, 33 % page, d - 1] = -inf
    layer, *_ = make(pkg, cuda, w, hq, 2, d, io)
    q = w.normal(2, hq, d, dtype=TYPES[io])
    q[0, 0], q[0, 2], q[1, 3], q[1, 5] = 0, 0, 0, 0  # (equal scores: weights that the type holds without a rest)
    out = layer.decode(q.view(2, -1).to(cuda), ints([n - 1] * 2, cuda), w.device_table(cuda)).view(2, hq, d).cpu()
    for b in range(2):
        exp, tol = ref.attend(q[b], w.keys, w.values, w.table[b], n - 1, page, d ** -0.5, out_type=TYPES[io], kept=w.kept)
        assert int((~exp.isfinite()).sum()) == hq // 2
        for h in range(hq):
            fine = exp[h].isfinite()
            assert torch.equal(out[b, h][~fine].float(), exp[h][~fine].float())
            close(out[b, h][fine], exp[h][fine], tol[h][fine], f"sequence {b}, head {h}")


@pytest.mark.parametrize("d,io,kept,page", FORMS)
@pytest.mark.parametrize("wide", [1, WIDE])
def test_decode_infinite_scores(pkg, cuda, d, io, kept, page, wide):
    """A key whose score is minus infinity takes no part; one whose score is infinity leaves no number."""
    n, hq, inf = 400, 6, float("inf")
    w = World([n] * 2, 2, d, page, kept, extra_width=wide)
    at = [(w.table[b][t // page], t % page) for b, t in ((0, n - 1), (1, 100))]
    layer, k, *_ = make(pkg, cuda, w, hq, 2, d, io)
    for (p, s), value in zip(at, (-inf, inf)):
        by_head(k, w.layout)[p, 0, s, 1] = value
    q = w.normal(2, hq, d, dtype=TYPES[io])
    q[:, :, 1] = 0.5  # the infinity's sign is the score's, and the type holds it without a rest
    out = layer.decode(q.view(2, -1).to(cuda), ints([n - 1] * 2, cuda), w.device_table(cuda)).view(2, hq, d)
    assert out[1, :3].isnan().all()
    exp, tol = ref.attend(q[1], w.keys, w.values, w.table[1], n - 1, page, d ** -0.5, out_type=TYPES[io], kept=w.kept)
    close(out[1, 3:], exp[3:], tol[3:])
    # sequence 0: the first kv head as if it ended one token earlier, the other with all tokens
    exp, tol = ref.attend(q[0], w.keys, w.values, w.table[0], n - 1, page, d ** -0.5, out_type=TYPES[io], kept=w.kept)
    close(out[0, 3:], exp[3:], tol[3:])
    exp, tol = ref.attend(q[0], w.keys, w.values, w.table[0], n - 2, page, d ** -0.5, out_type=TYPES[io], kept=w.kept)
    close(out[0, :3], exp[:3], tol[:3])


# ---------------------------------------------------------------- append: scaled and partial rotations
YARN = {"type": "yarn", "factor": 4.0, "original_context_length": 256.0, "beta_fast": 32.0, "beta_slow": 1.0}
ROTATIONS = [
    {"ropeScaling": YARN},
    {"ropeScaling": {**YARN, "attention_factor": 0.625}, "rotaryDim": 32},
    {"ropeScaling": {"type": "linear", "factor": 3.0}, "ropePairCount": 5},
    {"ropeScaling": {"type": "llama3", "factor": 8.0, "original_context_length": 64.0, "low_freq_factor": 1.0,
                     "high_freq_factor": 4.0}},
    {"ropeScaling": YARN, "ropePairCount": 9, "rotaryDim": 48},
    {"ropePairCount": 0},
    {"ropeFreqDim": 128, "rotaryDim": 40},
    {"ropeScaling": YARN, "ropeFreqDim": 512, "ropePairCount": 13, "norms": True},
]


@pytest.mark.parametrize("options", ROTATIONS, ids=lambda o: "-".join(sorted(o)))
@pytest.mark.parametrize("form", ["one", "chunks", "chunks without bounds"])
@pytest.mark.parametrize("d,io,kept", [(64, "fp16", "fp16"), (128, "bf16", "bf16"), (96, "fp32", "fp16"),
                                       (256, "fp32", "fp32"), (100, "fp32", "fp32"), (64, "fp32", "bf16")])
def test_append_scaled_and_partial_rotations(pkg, cuda, options, form, d, io, kept):
    """Every form of the append (block per row, rows, pages) turns the pairs below ropePairCount by the scaled
    frequencies, times the attention factor, and leaves the rest as it is."""
    o, hq, hk, page, theta = dict(options), 5, 5, 16, 10000.0
    norm = o.pop("norms", False)
    g = torch.Generator().manual_seed(1)
    qn, kn = (torch.randn(d, generator=g).mul(0.3).add(1) for _ in range(2))
    if norm:
        o["qNormWeight"], o["kNormWeight"] = qn.numpy(), kn.numpy()
    starts, chunks = [0, 17, 300], [1, 1, 1] if form == "one" else [40, 1, 33]
    w = World(starts, hk, d, page, kept, room=max(chunks))
    layer, k, v, bd = make(pkg, cuda, w, hq, hk, d, io, bounds=form != "chunks without bounds", ropeTheta=theta, **o)
    qkv = w.normal(sum(chunks), (hq + 2 * hk) * d, dtype=TYPES[io])
    offsets = None if form == "one" else ints([0, 40, 41, 74], cuda)
    query = layer.append(qkv.to(cuda), ints(starts, cuda), w.device_table(cuda), row_offsets=offsets).cpu()
    assert layer.context.error() == 0
    rotary = o.get("rotaryDim", d)
    inv, factor = oracle.rope_parameters(o.get("ropeFreqDim", rotary), theta, o.get("ropeScaling"))
    pairs = min(rotary // 2, o.get("ropePairCount", rotary // 2))
    turn = torch.as_tensor(inv[:pairs]).double()

    def rotated(x, pos):
        a, b = x[..., :pairs], x[..., rotary // 2:rotary // 2 + pairs]
        cos, sin = (pos * turn).cos(), (pos * turn).sin()
        y = x.clone()
        y[..., :pairs] = (a * cos - b * sin) * factor
        y[..., rotary // 2:rotary // 2 + pairs] = (b * cos + a * sin) * factor
        return y

    got_k, got_v, at = k.cpu(), v.cpu(), 0
    for b, n in enumerate(chunks):
        for i in range(n):
            x, pos = qkv[at].double().view(hq + 2 * hk, d), starts[b] + i
            q, kk = x[:hq], x[hq:hq + hk]
            if norm:
                q, kk = ref.rms(q, qn, 1e-6, False), ref.rms(kk, kn, 1e-6, False)
            q, kk = rotated(q, pos), rotated(kk, pos)
            p, slot = w.table[b][pos // page], pos % page
            close(query[at], q, ref.row_error(q, TYPES[io], d), f"query of sequence {b}, token {i}")
            close(got_k[p, :, slot], kk, ref.row_error(kk, w.kept, d), f"key of sequence {b}, token {i}")
            assert torch.equal(got_v[p, :, slot], x[hq + hk:].to(w.kept))
            at += 1


@pytest.mark.parametrize("d,kept", [(64, "fp32"), (128, "bf16"), (256, "fp32"), (100, "fp32")])
def test_append_chunks_at_far_positions(pkg, cuda, d, kept):
    """Angles of far positions are reduced in 64 bits, in the table of a page's slots too."""
    hq, hk, page, n, theta = 4, 2, 64, 150, 1e6
    start = (1 << 24) + 21
    first = start // page
    k, v = (torch.zeros(4, hk, page, d, dtype=TYPES[kept], device=cuda) for _ in range(2))
    bounds = torch.zeros(4, hk, 2, d, dtype=TYPES[kept], device=cuda)
    table = torch.full((1, first + 4), -1, dtype=torch.int32, device=cuda)
    table[0, first:] = ints([2, 0, 3, 1], cuda)
    layer = pkg.PagedAttention(hq * d, hq, 1 << 25, k, v, {"headDim": d, "kvHeadCount": hk, "ropeTheta": theta,
                                                           "dtype": torch.float32}, key_bounds=bounds)
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(n, (hq + 2 * hk) * d, generator=g)
    query = layer.append(qkv.to(cuda), ints([start], cuda), table, row_offsets=ints([0, n], cuda)).cpu()
    assert layer.context.error() == 0
    got = k.cpu()
    for i in range(n):
        q, kk, _ = ref.form_row(qkv[i], start + i, hq, hk, d, theta=theta)
        close(query[i], q, ref.row_error(q, torch.float32, d))
        close(got[(2, 0, 3, 1)[(start + i) // page - first], :, (start + i) % page], kk, ref.row_error(kk, TYPES[kept], d))


@pytest.mark.parametrize("options", [{"rotaryDim": 0}, {"rotaryDim": 16}, {"ropePairCount": 5}, {"rotaryDim": 24, "ropePairCount": 0}],
                         ids=str)
@pytest.mark.parametrize("form", ["one", "chunks", "chunks without bounds"])
@pytest.mark.parametrize("d,io,kept", [(64, "fp16", "fp16"), (128, "bf16", "bf16"), (96, "fp32", "fp16"), (256, "fp32", "fp32"),
                                       (100, "fp32", "fp32")])
def test_append_turns_only_the_pairs_it_should(pkg, cuda, options, form, d, io, kept):
    """An infinity or a NaN reaches its own dimension, and its pair's where that is turned, and no other."""
    hq, hk, page, starts, chunks = 2, 2, 16, [1, 17], [1, 1] if form == "one" else [40, 20]
    w = World(starts, hk, d, page, kept, room=40)
    layer, k, v, _ = make(pkg, cuda, w, hq, hk, d, io, bounds=form != "chunks without bounds", ropeTheta=1e4, **options)
    x = w.normal(sum(chunks), 3, hk, d, dtype=TYPES[io])
    for held in (float("inf"), float("-inf"), float("nan")):
        x[torch.rand(x.shape, generator=w.g) < 0.02] = held
    offsets = None if form == "one" else ints([0, 40, 60], cuda)
    query = layer.append(x.view(sum(chunks), -1).to(cuda), ints(starts, cuda), w.device_table(cuda), row_offsets=offsets)
    half = options.get("rotaryDim", d) // 2
    pairs = min(half, options.get("ropePairCount", half))
    hit = ~x.isfinite()
    both = hit[..., :pairs] | hit[..., half:half + pairs]
    hit[:, :2, :, :pairs], hit[:, :2, :, half:half + pairs] = both[:, :2], both[:, :2]
    still = torch.ones(d, dtype=torch.bool)
    still[:pairs] = still[half:half + pairs] = False
    assert torch.equal(~query.view(-1, hq, d).isfinite().cpu(), hit[:, 0])
    at = 0
    for b, n in enumerate(chunks):
        for i in range(n):
            p, slot = w.table[b][(starts[b] + i) // page], (starts[b] + i) % page
            for pool, part, plain in ((k, 1, still), (v, 2, torch.ones(d, dtype=torch.bool))):
                got, exp = pool[p, :, slot].cpu(), x[at, part]
                assert torch.equal(~got.isfinite(), hit[at, part])
                assert torch.equal(got[:, plain].nan_to_num(nan=77.0), exp[:, plain].to(w.kept).nan_to_num(nan=77.0))
            at += 1


# ---------------------------------------------------------------- gates, alignment, empty calls
@pytest.mark.parametrize("d,io,kept,page", [(64, "fp32", "fp32", 16), (128, "fp32", "bf16", 16), (64, "fp16", "fp16", 4),
                                            (100, "fp16", "fp16", 16), (256, "fp32", "fp16", 16)])
@pytest.mark.parametrize("wide", [1, WIDE])
def test_decode_gate_as_output_everywhere(pkg, cuda, d, io, kept, page, wide):
    """The gate's own memory as the output, for the kernels that join many shares and those that do not."""
    w = World([700, 40, 0], 2, d, page, kept, extra_width=wide)
    layer, *_ = make(pkg, cuda, w, 8, 2, d, io)
    q, gate = (w.normal(3, 8 * d, dtype=TYPES[io]).to(cuda) for _ in range(2))
    pos, table = ints([699, 39, -1], cuda), w.device_table(cuda)
    exp = layer.decode(q, pos, table, gate=gate)
    assert torch.equal(layer.decode(q, pos, table, gate=gate, out=gate), exp)


@pytest.mark.parametrize("d,io,kept,page", [(64, "fp16", "fp16", 16), (128, "bf16", "bf16", 16), (64, "fp32", "fp16", 32),
                                            (64, "fp32", "fp32", 16), (128, "fp32", "bf16", 16), (64, "fp16", "fp16", 4),
                                            (100, "fp16", "fp16", 16), (256, "fp32", "fp16", 16)])
@pytest.mark.parametrize("wide", [1, WIDE])
@pytest.mark.parametrize("held", [0.0, float("inf"), float("-inf"), float("nan")])
def test_decode_zeros_whatever_the_gate_holds(pkg, cuda, d, io, kept, page, wide, held):
    """Rows with nothing to attend to (no sequence, a position past the capacity, an empty list, no page that is in
    the pool) are zeros also where the gate has no number."""
    w = World([700, 0, 40, 40], 2, d, page, kept, extra_width=wide)
    layer, *_ = make(pkg, cuda, w, 8, 2, d, io)
    q, gate = (w.normal(4, 8 * d, dtype=TYPES[io]).to(cuda) for _ in range(2))
    gate[1:] = held
    table = w.device_table(cuda)
    table[3] = -7
    out = layer.decode(q, ints([699, -1, w.width * page, 39], cuda), table, gate=gate)
    assert not out[1:].any() and out[0].isfinite().all() and out[0].any()
    pages = ints([[[0, 1], [1, -1]]] + [[[-1, -1], [-1, -1]]] * 3, cuda)
    out = layer.decode(q, ints([699, -1, 39, 39], cuda), w.device_table(cuda), pages=pages, gate=gate)
    assert not out[1:].any() and out[0].isfinite().all() and out[0].any()
    layer.context.error()


@pytest.mark.parametrize("io,kept", PAIRS)
def test_rows_off_the_16_byte_boundaries(pkg, cuda, io, kept):
    """A head_dim that is no multiple of 8: any row of a tensor may be the first one."""
    d, page = 101, 8
    w = World([30, 77], 1, d, page, kept, room=1)
    layer, k, v, bd = make(pkg, cuda, w, 1, 1, d, io, rotaryDim=0)
    q, gate, qkv = (w.normal(3, n * d, dtype=TYPES[io]).to(cuda) for n in (1, 1, 3))
    pos, table = ints([29, 76], cuda), w.device_table(cuda)
    out = torch.full((3, d), 7.0, dtype=TYPES[io], device=cuda)
    layer.decode(q[1:], pos, table, gate=gate[1:], out=out[1:])
    assert torch.equal(out[1:], layer.decode(q[1:].clone(), pos, table, gate=gate[1:].clone()))
    assert (out[0] == 7).all()
    assert torch.equal(layer.select(q[1:], pos, table, 3), layer.select(q[1:].clone(), pos, table, 3))
    query = torch.full((3, d), 7.0, dtype=TYPES[io], device=cuda)
    layer.append(qkv[1:], pos + 1, table, query=query[1:])
    assert layer.context.error() == 0
    assert torch.equal(query[1:], qkv[1:, :d]) and (query[0] == 7).all()
    for b, n in enumerate((30, 77)):
        at = w.table[b][n // page], 0, n % page
        assert torch.equal(k[at], qkv[1 + b, d:2 * d].to(w.kept)) and torch.equal(v[at], qkv[1 + b, 2 * d:].to(w.kept))


def test_unaligned_addresses_of_vector_kernels_are_refused(pkg, cuda):
    w = World([30], 1, 64, 16, "fp16")
    layer, *_ = make(pkg, cuda, w, 1, 1, 64, "fp16")
    buf = torch.zeros(1024, dtype=torch.float16, device=cuda)
    pos, table, row = ints([29], cuda), w.device_table(cuda), torch.zeros(1, 64, dtype=torch.float16, device=cuda)
    off, whole = buf[4:68].view(1, 64), buf[4:196].view(1, 192)
    for call in (lambda: layer.decode(off, pos, table), lambda: layer.decode(row, pos, table, out=off),
                 lambda: layer.decode(row, pos, table, gate=off), lambda: layer.append(whole, pos, table),
                 lambda: layer.select(off, pos, table, 2),
                 lambda: layer.append(buf[:192].view(1, 192), pos, table, query=buf[260:324].view(1, 64))):
        with pytest.raises(pkg.TlaError, match="INVALID_ARG"):
            call()
    # half an element, through the C ABI
    odd = make(pkg, cuda, World([30], 1, 101, 16, "fp16"), 1, 1, 101, "fp16", rotaryDim=0)[0]
    assert pkg.lib().tla_paged_decode(odd.handle, buf.data_ptr() + 1, pos.data_ptr(), table.data_ptr(), w.width, None, 0,
                                      None, buf.data_ptr() + 512, 1, None, 0, None) == -1


def test_an_empty_batch_with_a_page_list(pkg, cuda):
    """No sequences: nothing to do, with or without lists."""
    layer = make(pkg, cuda, World([30], 2, 64, 16, "fp16"), 8, 2, 64, "fp16")[0]
    q, none = torch.zeros(0, 512, dtype=torch.float16, device=cuda), ints([], cuda)
    table = torch.zeros(0, 3, dtype=torch.int32, device=cuda)
    pages = layer.select(q, none, table, 5)
    assert pages.shape == (0, 2, 5)
    assert layer.decode(q, none, table, pages=pages).shape == (0, 512)


# ---------------------------------------------------------------- append: offsets out of order, inside guarded buffers
@pytest.mark.parametrize("d,io,kept", [(64, "fp16", "fp16"), (128, "fp32", "bf16"), (100, "fp16", "fp16"), (256, "fp32", "fp32")])
@pytest.mark.parametrize("bounded", [True, False])
@pytest.mark.parametrize("offsets", [[0, 30, 5, 20], [5, 3, 1, 0], [0, 0, 0, 1 << 30], [-(1 << 31), 4, 9, 20],
                                     [-5, -3, 2, 18], [20, 20, 20, 20], [0, 20, 0, 20], [(1 << 31) - 1, 0, -(1 << 31), 7]])
def test_append_offsets_out_of_order_touch_nothing_else(pkg, cuda, d, io, kept, bounded, offsets):
    """Rows may move or be lost, but what surrounds the rows is neither read nor written, nor is any page that the
    table does not name."""
    w = World([0, 0, 0], 2, d, 16, kept, room=32)
    guard = 4096

    def inside(shape, dtype, fill):
        n = math.prod(shape)
        whole = torch.full((n + 2 * guard,), fill, dtype=dtype, device=cuda)
        return whole, whole[guard:guard + n].view(shape)

    pages = w.keys.shape[0]
    kw, k = inside((pages, 2, 16, d), w.kept, 3.0)
    vw, v = inside((pages, 2, 16, d), w.kept, 3.0)
    bw, bd = inside((pages, 2, 2, d), w.kept, 3.0)
    xw, x = inside((20, 8 * d), TYPES[io], float("nan"))
    qw, query = inside((20, 4 * d), TYPES[io], 3.0)
    x.copy_(w.normal(20, 8 * d, dtype=TYPES[io]).clamp(-2, 2))
    layer = pkg.PagedAttention(4 * d, 4, w.width * 16, k, v, {"headDim": d, "kvHeadCount": 2, "dtype": TYPES[io]},
                               key_bounds=bd if bounded else None)
    layer.append(x, ints([0, 7, 16], cuda), w.device_table(cuda), row_offsets=ints(offsets, cuda), query=query)
    assert layer.context.error() != -17
    named = sorted({p for row in w.table for p in row if p >= 0})
    spare = [p for p in range(pages) if p not in named]
    for whole, inner in ((kw, k), (vw, v), (bw, bd), (qw, query)):
        assert (whole[:guard] == 3).all() and (whole[-guard:] == 3).all()
        assert inner.isfinite().all()  # (a row from outside would be NaN)
    for t in (k, v, bd):
        assert (t[spare] == 3).all()
    if not bounded:
        assert (bw == 3).all()


def test_edges_under_bounds_check_build(pkg):
    """These tests in a fresh process that loads libtla_check.so: no guarded index may leave its buffer."""
    if os.environ.get("TLA_LIBRARY"):
        pytest.skip("runs in that process")
    subprocess.run(["make", "-s", "-j8", "-C", str(ROOT / "three-llm_b200" / "csrc"), "check"], check=True)
    env = dict(os.environ, TLA_LIBRARY=str(ROOT / "three-llm_b200" / "libtla_check.so"))
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-p", "no:cacheprovider", "-m", "gpu",
                        "tests/test_paged_edges_gpu.py"], cwd=ROOT, env=env, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-2000:]
    assert " passed" in r.stdout
