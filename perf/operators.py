"""Operators of the paged key-value cache: their cases, plain forms and calls.

Three operators share a pool of fixed-size pages, [pages][kv heads][slots][d]
("HND") or [pages][slots][kv heads][d] ("NHD"), and a page table that lists
each sequence's pages in order:

  append  rows of [Q | K | V] get their QK-norm and rotation; the keys and
          values go to their pages' slots, the rotated queries come back, and
          each touched page's bounds (the smallest and largest key value per
          head and dimension) take the new keys in.
  decode  attention of one new token per sequence over its pages.
  sparse  the same over the pages that a cheap score selects: the sum over a
          kv head's query heads of the upper bound that a page's key bounds
          set on its dot products, formed in 64 bits and rounded to 32; ties
          go to the lowest page. The first and the last page always take part.

`run` computes them with elementary torch operations, or where `own` is true
through the package's PagedAttention.
"""
import importlib
import math
import random

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_EPS = 1e-6  # of the QK-norm
_SPARE = 5   # pages of a pool that no sequence holds


def _case(name, op, batch, tokens, spread, hq, hk, d, page, layout="HND", io="fp16", pages="fp16", theta=500000.0,
          rotary=0, norm=False, chunk=0, window=0, gate=False, unused=0, count=0):
    """tokens: the longest sequence's length after the call; spread: "equal", or "ragged" for lengths spread over
    their logarithm below it. chunk (append): the most new tokens of a sequence, 0 for one token each. unused
    (decode): rows of the batch without a sequence. count (sparse): pages that take part. rotary 0: all of d."""
    return {"name": name, "op": op, "batch": batch, "tokens": tokens, "spread": spread, "hq": hq, "hk": hk, "d": d,
            "page": page, "layout": layout, "io": io, "pages": pages, "theta": theta, "rotary": rotary, "norm": norm,
            "chunk": chunk, "window": window, "gate": gate, "unused": unused, "count": count}


def listed():
    return [
        # the token that a single short chat appends: the smallest call there is, all latency
        _case("append one token", "append", 1, 129, "equal", 8, 2, 64, 16, theta=10000.0),
        # one decode step of a full serving batch of a 1B-class model, 4096 tokens cached
        _case("append 64 tokens", "append", 64, 4097, "equal", 32, 8, 64, 16),
        # a prompt of a 0.5B-class model, appended from its start
        _case("append a prompt", "append", 1, 2048, "equal", 14, 2, 64, 64, theta=1000000.0, chunk=2048),
        # chunks of 16 prompts of an 8B-class model with QK-norm, most starting inside a page
        _case("append ragged chunks", "append", 16, 8192, "ragged", 32, 8, 128, 64, "NHD", "bf16", "bf16", norm=True,
              chunk=2047),
        # the step of a single short chat
        _case("decode one short", "decode", 1, 129, "equal", 8, 2, 64, 16, theta=10000.0),
        # eight users of a 1B-class model at 4096 tokens
        _case("decode 8 x 4097", "decode", 8, 4097, "equal", 32, 8, 64, 16),
        # a serving batch of an 8B-class model, lengths from hundreds to thousands
        _case("decode 64 ragged", "decode", 64, 8192, "ragged", 32, 8, 128, 64, "NHD", "bf16", "bf16"),
        # one long document
        _case("decode one of 131072", "decode", 1, 131072, "equal", 32, 8, 128, 64),
        # layers with a sliding window and an output gate, float32 activations, a batch padded to a captured size
        _case("decode windowed fp32", "decode", 24, 6001, "ragged", 14, 2, 64, 32, io="fp32", theta=1000000.0,
              window=1000, gate=True, unused=3),
        # the smallest cache where choosing pages pays: half of 64 pages
        _case("sparse one of 1024", "sparse", 1, 1024, "equal", 32, 8, 64, 16, count=32),
        # one long document, 1/32 of its pages read
        _case("sparse one of 131072", "sparse", 1, 131072, "equal", 32, 8, 128, 64, count=64),
        # a batch of long conversations
        _case("sparse 32 ragged", "sparse", 32, 16384, "ragged", 32, 8, 128, 64, io="bf16", pages="bf16", count=48),
    ]


def draw(rng):
    """Batches from 1 to 64, sequences of 1 to 131072 tokens, chunks to 2048, within the largest listed case's work."""
    most = max(work(c)["bytes"] for c in listed())

    def spread(lo, hi):
        return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))

    while True:
        op = rng.choice(["append", "decode", "sparse"])
        hq, hk = rng.choice([(8, 2), (14, 2), (32, 8), (16, 16), (16, 1), (12, 4)])
        d = rng.choice([64, 128])
        kind = rng.choice(["fp16", "bf16", "fp32"])
        page = rng.choice([16, 32, 64, 128])
        c = _case("", op, spread(1, 64), 0, rng.choice(["equal", "ragged"]), hq, hk, d, page,
                  rng.choice(["HND", "NHD"]), kind, "fp16" if kind == "fp32" else kind,
                  rng.choice([10000.0, 500000.0, 1000000.0]))
        del c["name"]
        if op == "append":
            c["chunk"] = rng.choice([0, spread(1, 2048)])
            c["tokens"] = max(1, c["chunk"]) + spread(1, 16384) - 1
            c["rotary"] = rng.choice([0, d // 2])
            c["norm"] = rng.random() < 0.5
        elif op == "decode":
            c["tokens"] = spread(1, 131072)
            c["window"] = rng.choice([0, 0, spread(1, 4096)])
            c["gate"] = rng.random() < 0.3
            c["unused"] = rng.choice([0, 0, c["batch"] // 4])
        else:
            c["tokens"] = spread(64, 131072)
            c["count"] = spread(4, 128)
        held = c["batch"] * c["tokens"] * hk * d * 4  # bytes of the pool, about: three states fit with room
        if held <= 6 << 30 and work(c)["bytes"] <= most:
            return c


def _lengths(case):
    """Each sequence's length after the call (the case's own, whatever the seed)."""
    n, top = case["batch"], case["tokens"]
    if case["spread"] == "equal":
        return [top] * n
    r = random.Random(17)
    low = max(1, top // 16, case["chunk"])
    return [top] + [min(top, int(math.exp(r.uniform(math.log(low), math.log(top + 1))))) for _ in range(n - 1)]


def _chunks(case, lengths):
    """New tokens of each sequence (append)."""
    if not case["chunk"]:
        return [1] * len(lengths)
    if case["spread"] == "equal":
        return [min(case["chunk"], n) for n in lengths]
    r = random.Random(5)
    return [min(case["chunk"], lengths[0])] + [min(n, r.randint(1, case["chunk"])) for n in lengths[1:]]


def prepare(case, seed):
    lengths = _lengths(case)
    page, hq, hk, d, batch = case["page"], case["hq"], case["hk"], case["d"], case["batch"]
    io, kept = _TYPES[case["io"]], _TYPES[case["pages"]]
    g = torch.Generator("cuda").manual_seed(seed)
    held = [-(-n // page) for n in lengths]
    width, total = max(held), sum(held) + _SPARE
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    table, at = [], 0
    for n in held:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    s = {"case": dict(case), "lengths": lengths, "table": torch.tensor(table, dtype=torch.int32).cuda()}
    shape = (total, hk, page, d) if case["layout"] == "HND" else (total, page, hk, d)
    slot_dim = 2 if case["layout"] == "HND" else 1
    about = tuple(1 if i == slot_dim else n for i, n in enumerate(shape))
    # keys gather around a direction of their page, as neighbouring tokens' keys do
    keys = torch.empty(shape, dtype=kept, device="cuda").normal_(generator=g)
    keys.mul_(0.8).add_(torch.empty(about, dtype=kept, device="cuda").normal_(generator=g), alpha=0.6)
    s["keys"] = keys
    s["values"] = torch.empty(shape, dtype=kept, device="cuda").normal_(generator=g)
    if case["op"] == "append":
        new = _chunks(case, lengths)
        starts = [n - c for n, c in zip(lengths, new)]
        s["starts"] = torch.tensor(starts, dtype=torch.int32).cuda()
        s["offsets"] = None
        if case["chunk"]:
            ends = [0]
            for c in new:
                ends.append(ends[-1] + c)
            s["offsets"] = torch.tensor(ends, dtype=torch.int32).cuda()
        s["most_pages"] = max((n - 1) // page - b // page + 1 for n, b in zip(lengths, starts))
        s["qkv"] = torch.randn((sum(new), (hq + 2 * hk) * d), generator=g, device="cuda").to(io)
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            r = random.Random(seed)
            s["q_norm"] = [1 + 0.1 * r.gauss(0, 1) for _ in range(d)]
            s["k_norm"] = [1 + 0.1 * r.gauss(0, 1) for _ in range(d)]
        # before the call the bounds hold the tokens that are there already
        s["bounds"] = _bounds_of(s["keys"], s["table"], s["starts"], case)
    else:
        s["positions"] = torch.tensor([n - 1 for n in lengths], dtype=torch.int32).cuda()
        if case["unused"]:
            s["positions"][-case["unused"]:] = -1
        s["query"] = torch.randn((batch, hq * d), generator=g, device="cuda").to(io)
        s["gate"] = torch.randn((batch, hq * d), generator=g, device="cuda").to(io) if case["gate"] else None
        s["bounds"] = None
        if case["op"] == "sparse":
            s["bounds"] = _bounds_of(s["keys"], s["table"], s["positions"] + 1, case)
    if own:
        s["layer"] = _layer(s)
    return s


def _bounds_of(keys, table, lengths, case):
    """[pages][kv heads][2][d]: the smallest and largest key per page over its first slots, as the lengths fill them."""
    page, k = case["page"], keys if case["layout"] == "HND" else keys.transpose(1, 2)
    filled = torch.zeros(k.shape[0] + 1, dtype=torch.int64, device=k.device)
    first = torch.arange(table.shape[1], device=k.device) * page
    n = (lengths[:, None] - first[None, :]).clamp(0, page)
    filled[torch.where(table < 0, k.shape[0], table).long().reshape(-1)] = n.reshape(-1)
    empty = torch.arange(page, device=k.device)[None, :] >= filled[:-1, None]
    low = k.masked_fill(empty[:, None, :, None], math.inf).amin(2)
    high = k.masked_fill(empty[:, None, :, None], -math.inf).amax(2)
    none = (filled[:-1] == 0)[:, None, None]
    return torch.stack((low.masked_fill(none, 0), high.masked_fill(none, 0)), 2).contiguous()


def _layer(s):
    package, c = importlib.import_module("three-llm_b200"), s["case"]
    options = {"headDim": c["d"], "kvHeadCount": c["hk"], "ropeTheta": c["theta"], "maxBatch": c["batch"],
               "dtype": _TYPES[c["io"]], "pageLayout": c["layout"], "slidingWindow": c["window"], "rmsEpsilon": _EPS,
               "qNormWeight": s.get("q_norm"), "kNormWeight": s.get("k_norm")}
    if c["rotary"]:
        options["rotaryDim"] = c["rotary"]
    return package.PagedAttention(c["hq"] * c["d"], c["hq"], s["table"].shape[1] * c["page"], s["keys"], s["values"],
                                  options, key_bounds=s["bounds"])


def run(s):
    op = s["case"]["op"]
    if own:
        layer = s["layer"]
        if op == "append":
            query = layer.append(s["qkv"], s["starts"], s["table"], row_offsets=s["offsets"])
            return {"query": query, "keys": s["keys"], "values": s["values"], "bounds": s["bounds"]}
        if op == "decode":
            return {"out": layer.decode(s["query"], s["positions"], s["table"], gate=s["gate"])}
        pages = layer.select(s["query"], s["positions"], s["table"], s["case"]["count"])
        return {"pages": pages, "out": layer.decode(s["query"], s["positions"], s["table"], pages=pages)}
    return {"append": _append, "decode": _decode, "sparse": _sparse}[op](s)


# ---------------------------------------------------------------- plain forms
def _rms(x, weight):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * torch.tensor(weight, device=x.device)


def _frequencies(case, device):
    """As rope_parameters gives them: 1 / theta^(2 i / r) in 64 bits, held in float32."""
    r = case["rotary"] or case["d"]
    return (1 / case["theta"] ** (torch.arange(0, r, 2, dtype=torch.float64, device=device) / r)).float()


def _rotate(x, positions, case):
    """x [n][heads][d] float32; pair i of the rotary dimensions is (i, i + r / 2)."""
    f = _frequencies(case, x.device)
    angle = positions.double()[:, None] * f.double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    h = f.numel()
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * h:]), -1)


def _append(s):
    c, keys, values, bounds = s["case"], s["keys"], s["values"], s["bounds"]
    hq, hk, d, page = c["hq"], c["hk"], c["d"], c["page"]
    n, dev = s["qkv"].shape[0], keys.device
    token = torch.arange(n, device=dev)
    if s["offsets"] is None:
        row, position, last = token, s["starts"].long(), s["starts"].long()
    else:
        off = s["offsets"].long()
        row = torch.searchsorted(off, token, right=True) - 1
        position = s["starts"].long()[row] + token - off[row]
        last = s["starts"].long() + off[1:] - off[:-1] - 1
    x = s["qkv"].float().view(n, hq + 2 * hk, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    if c["norm"]:
        q, k = _rms(q, s["q_norm"]), _rms(k, s["k_norm"])
    q, k = _rotate(q, position, c), _rotate(k, position, c)
    at, slot = s["table"].long()[row, position // page], position % page
    kp, vp = (keys, values) if c["layout"] == "HND" else (keys.transpose(1, 2), values.transpose(1, 2))
    kp[at, :, slot] = k.to(keys.dtype)
    vp[at, :, slot] = v.to(values.dtype)
    # the touched pages' bounds, over the slots that are filled now
    first = s["starts"].long() // page
    logical = torch.minimum(first[:, None] + torch.arange(s["most_pages"], device=dev), (last // page)[:, None])
    touched = s["table"].long().gather(1, logical)
    filled = (last[:, None] - logical * page + 1).clamp(max=page).reshape(-1)
    empty = (torch.arange(page, device=dev)[None] >= filled[:, None])[:, None, :, None]
    held = kp[touched.reshape(-1)]
    bounds[touched.reshape(-1)] = torch.stack((held.masked_fill(empty, math.inf).amin(2),
                                               held.masked_fill(empty, -math.inf).amax(2)), 2)
    return {"query": q.reshape(n, hq * d).to(s["qkv"].dtype), "keys": keys, "values": values, "bounds": bounds}


def _attend(s, k, v, token, seen):
    """k, v [B][kv heads][n][d] in 32 bits, seen [B][1 or kv heads][n]: which of them take part."""
    c = s["case"]
    b, hk, g, d = k.shape[0], c["hk"], c["hq"] // c["hk"], c["d"]
    score = torch.matmul(s["query"].float().view(b, hk, g, d), k.transpose(2, 3)) / math.sqrt(d)
    score = score.masked_fill(~seen[:, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w, v) / torch.where(total == 0, 1.0, total)
    out = out.reshape(b, hk * g * d)
    if s["gate"] is not None:
        out = out / (1 + torch.exp(-s["gate"].float()))
    return out.to(s["query"].dtype)


def _decode(s):
    c, table = s["case"], s["table"].long().clamp(min=0)
    kp, vp = (s["keys"], s["values"]) if c["layout"] == "HND" else (s["keys"].transpose(1, 2), s["values"].transpose(1, 2))
    b, hk, d = c["batch"], c["hk"], c["d"]
    k = kp[table].transpose(1, 2).reshape(b, hk, -1, d).float()
    v = vp[table].transpose(1, 2).reshape(b, hk, -1, d).float()
    token = torch.arange(k.shape[2], device=k.device)[None]
    position = s["positions"].long()[:, None]
    seen = token <= position
    if c["window"]:
        seen &= token > position - c["window"]
    return {"out": _attend(s, k, v, token, seen[:, None])}


def _selected(s):
    """[B][kv heads][count] int32: the pages that take part, in their order, then -1."""
    c, table = s["case"], s["table"].long()
    b, hk, g, d, page = c["batch"], c["hk"], c["hq"] // c["hk"], c["d"], c["page"]
    q = s["query"].double().view(b, hk, g, d)
    up, down = q.clamp(min=0).sum(2), q.clamp(max=0).sum(2)
    held = s["bounds"][table.clamp(min=0)].double()  # [B][pages][kv heads][2][d]
    score = torch.einsum("bphd,bhd->bhp", held[:, :, :, 1], up) + torch.einsum("bphd,bhd->bhp", held[:, :, :, 0], down)
    score = score.float() + 0.0
    n = s["positions"].long() // page + 1
    at = torch.arange(table.shape[1], device=table.device)
    always = (at < 1) | (at[None] == n[:, None] - 1)
    score = score.masked_fill(always[:, None], math.inf)
    score = score.masked_fill((at[None] >= n[:, None])[:, None], -math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :c["count"]]
    best = best.masked_fill(best >= n[:, None, None], table.shape[1])
    best = torch.sort(best, dim=-1).values
    out = torch.full((b, hk, c["count"]), -1, dtype=torch.int32, device=table.device)
    out[..., :best.shape[-1]] = torch.where(best == table.shape[1], -1, best).int()
    return out


def _sparse(s):
    c, table, pages = s["case"], s["table"].long(), _selected(s)
    b, hk, d, page, count = c["batch"], c["hk"], c["d"], c["page"], c["count"]
    kp, vp = (s["keys"], s["values"]) if c["layout"] == "HND" else (s["keys"].transpose(1, 2), s["values"].transpose(1, 2))
    logical = pages.long().clamp(min=0)
    at = table[:, None].expand(-1, hk, -1).gather(2, logical).clamp(min=0)
    head = torch.arange(hk, device=table.device)[None, :, None]
    k = kp[at, head].reshape(b, hk, count * page, d).float()
    v = vp[at, head].reshape(b, hk, count * page, d).float()
    token = (logical[..., None] * page + torch.arange(page, device=table.device)).reshape(b, hk, -1)
    seen = (token <= s["positions"].long()[:, None, None]) & (pages >= 0).repeat_interleave(page, 2)
    return {"pages": pages, "out": _attend(s, k, v, token, seen)}


# ---------------------------------------------------------------- what a pass cannot do without
def _attended(case, lengths):
    seen = [n if not case["window"] else min(n, case["window"]) for n in lengths]
    if case["unused"]:
        seen = seen[:-case["unused"]]
    if case["op"] == "sparse":
        seen = [min(n, case["count"] * case["page"] - case["page"] + (n - 1) % case["page"] + 1) for n in seen]
    return sum(seen)


def work(case):
    lengths = _lengths(case)
    hq, hk, d, page = case["hq"], case["hk"], case["d"], case["page"]
    io, kept = (4 if case[t] == "fp32" else 2 for t in ("io", "pages"))
    if case["op"] == "append":
        new = _chunks(case, lengths)
        n = sum(new)
        touched = sum((e - 1) // page - (e - c) // page + 1 for e, c in zip(lengths, new))
        partly = sum((e - c) % page != 0 for e, c in zip(lengths, new))  # bounds that are read too
        return {"bytes": n * ((2 * hq + 2 * hk) * io + 2 * hk * kept) * d + (touched + partly) * hk * 2 * d * kept,
                "flops": n * (hq + hk) * 3 * d}
    tokens, rows = _attended(case, lengths), case["batch"]
    moved = tokens * 2 * hk * d * kept + rows * hq * d * io * (3 if case["gate"] else 2)
    flops = 4 * tokens * hq * d
    if case["op"] == "sparse":
        pages = sum(-(-n // page) for n in lengths)
        moved += pages * hk * 2 * d * kept + rows * hk * case["count"] * 4
        flops += 4 * pages * hk * d
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    global own
    as_set, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = as_set
    c, f64 = case, torch.float64
    hq, hk, d, page = c["hq"], c["hk"], c["d"], c["page"]
    g, dev, table = hq // hk, s["keys"].device, s["table"].tolist()
    by_head = c["layout"] == "HND"
    if c["op"] == "append":
        keys, values, bounds = s["keys"].to(f64), s["values"].to(f64), s["bounds"].to(f64)
        query = torch.empty((s["qkv"].shape[0], hq, d), dtype=f64, device=dev)
        r = c["rotary"] or d
        turn = torch.tensor([c["theta"] ** (-2.0 * i / r) for i in range(r // 2)], dtype=torch.float32).to(dev, f64)
        begin = 0
        for b, n in enumerate(_chunks(c, s["lengths"])):
            x = s["qkv"][begin:begin + n].to(f64).view(n, hq + 2 * hk, d)
            start = s["lengths"][b] - n
            qk = x[:, :hq + hk].clone()
            if c["norm"]:
                scale = torch.stack([torch.tensor(s["q_norm"], dtype=torch.float32).to(dev, f64)] * hq
                                    + [torch.tensor(s["k_norm"], dtype=torch.float32).to(dev, f64)] * hk)
                qk = qk / ((qk * qk).sum(-1, keepdim=True) / d + _EPS).sqrt() * scale
            angle = torch.outer(torch.arange(start, start + n, device=dev).to(f64), turn)
            z = torch.polar(torch.ones_like(angle), angle)[:, None] * torch.complex(qk[..., :r // 2].contiguous(), qk[..., r // 2:r].contiguous())
            qk[..., :r // 2], qk[..., r // 2:r] = z.real, z.imag
            query[begin:begin + n] = qk[:, :hq]
            done = 0
            while done < n:
                at = start + done
                p, slot = table[b][at // page], at % page
                m = min(page - slot, n - done)
                k, v = qk[done:done + m, hq:], x[done:done + m, hq + hk:]
                if by_head:
                    keys[p, :, slot:slot + m], values[p, :, slot:slot + m] = k.transpose(0, 1), v.transpose(0, 1)
                else:
                    keys[p, slot:slot + m], values[p, slot:slot + m] = k, v
                low, high = k.min(0).values, k.max(0).values
                if slot:
                    low, high = torch.minimum(low, bounds[p, :, 0]), torch.maximum(high, bounds[p, :, 1])
                bounds[p, :, 0], bounds[p, :, 1] = low, high
                done += m
            begin += n
        return {"query": query.reshape(-1, hq * d), "keys": keys, "values": values, "bounds": bounds}
    out = torch.zeros((c["batch"], hq, d), dtype=f64, device=dev)
    chosen = torch.full((c["batch"], hk, max(1, c["count"])), -1, dtype=torch.int32, device=dev)
    for b, position in enumerate(s["positions"].tolist()):
        if position < 0:
            continue
        first = max(0, position - c["window"] + 1) if c["window"] else 0
        held = torch.tensor(table[b][:position // page + 1], device=dev)
        q = s["query"][b].to(f64).view(hk, g, d)
        if c["op"] == "sparse" and len(held) > c["count"]:
            low, high = s["bounds"][held, :, 0].to(f64), s["bounds"][held, :, 1].to(f64)
            bound = torch.zeros((len(held), hk), dtype=f64, device=dev)
            for i in range(g):
                bound += torch.maximum(q[None, :, i] * low, q[None, :, i] * high).sum(-1)
            bound = bound.float()
            bound[0], bound[-1] = math.inf, math.inf
            kept = torch.sort(torch.argsort(bound, dim=0, descending=True, stable=True)[:c["count"]], dim=0).values.t()
        else:
            kept = torch.arange(len(held), device=dev).expand(hk, -1)
        if c["op"] == "sparse":
            chosen[b, :, :kept.shape[1]] = kept.int()
        for h in range(hk):
            at = held[kept[h]]
            k = (s["keys"][at, h] if by_head else s["keys"][at, :, h]).reshape(-1, d).to(f64)
            v = (s["values"][at, h] if by_head else s["values"][at, :, h]).reshape(-1, d).to(f64)
            where = (kept[h][:, None] * page + torch.arange(page, device=dev)).reshape(-1)
            use = (where <= position) & (where >= first)
            w = torch.softmax(q[h] @ k[use].t() / d ** 0.5, -1)
            out[b, h * g:(h + 1) * g] = w @ v[use]
    out = out.reshape(c["batch"], hq * d)
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].to(f64))
    return {"pages": chosen, "out": out} if c["op"] == "sparse" else {"out": out}
