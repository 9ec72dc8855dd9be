"""The paged cache's operators in 64 bits on the host, with the error that the
kernels' roundings may add to each output.

A pool is a torch tensor [pages][kv heads][slots][d] of the pages' type on the
host; tables, positions and lists are plain lists. Nothing here is shared with
the package.
"""
import math

import torch

F64 = torch.float64


def half_step(dtype):
    """A rounding to dtype is off by at most this much, relative to the value."""
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the spacing of dtype's smallest values: the error of a rounding near zero."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def frequencies(theta, rotary):
    """1 / theta^(2 i / rotary), held in float32 (rope.ts:4-52)."""
    return torch.tensor([theta ** (-2.0 * i / rotary) for i in range(rotary // 2)], dtype=F64).float().to(F64)


def rms(x, weight, eps, offset):
    w = torch.ones(x.shape[-1], dtype=F64) if weight is None else torch.as_tensor(weight).float().to(F64)
    if offset and weight is not None:
        w = 1 + w
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w


def rotate(x, position, theta, rotary):
    if not theta or not rotary:
        return x
    angle = position * frequencies(theta, rotary)
    h = rotary // 2
    a, b = x[..., :h], x[..., h:rotary]
    return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), x[..., rotary:]), -1)


def form_row(row, position, hq, hk, d, theta=0.0, rotary=None, q_norm=None, k_norm=None, eps=1e-6, offset=False,
             v_norm=False):
    """(q, k, v) of one [Q | K | V] row at a position, in 64 bits."""
    x = row.to(F64).view(hq + 2 * hk, d)
    q, k, v = x[:hq], x[hq:hq + hk], x[hq + hk:]
    if q_norm is not None:
        q = rms(q, q_norm, eps, offset)
    if k_norm is not None:
        k = rms(k, k_norm, eps, offset)
    if v_norm:
        v = rms(v, None, eps, False)
    rotary = d if rotary is None else rotary
    return rotate(q, position, theta, rotary), rotate(k, position, theta, rotary), v


def row_error(x, dtype, d):
    """What forming a value of size |x| (norm, sine, cosine and the rotation in 32 bits) and rounding it to
    dtype may be off by. 32-bit: the sum of squares d 2^-24, ten roundings and the 2 ulp of sincosf after a
    reduction in 64 bits; the rotation adds two products, each at most the pair's size, so the pair's larger
    size (at most the head's largest) carries the error."""
    size = x.abs().amax(-1, keepdim=True)
    return half_step(dtype) * x.abs() + (d + 16) * 2.0 ** -24 * 2 * size + smallest(dtype)


def attend(q, keys, values, table, position, page, scale, window=0, listed=None, gate=None, out_type=torch.float16,
           kept=torch.float16, bad=()):
    """(out, error bound) of one sequence: q [hq][d], keys / values the pool, listed[kvh] the page indexes or
    None; `bad` pages of the pool's range are skipped when the table names something else.

    The bound: P is rounded to the pages' 16-bit type before P V (half a step of each weight, or half the
    smallest spacing), the output once to out_type; the dot products and sums run in 32 bits (d + 8
    roundings of a score's absolute sum, n + 64 of the output's). With float32 activations or pages nothing
    is rounded to 16 bits but split in two parts, 2^-22 of each product at most."""
    hk, d = keys.shape[1], keys.shape[3]
    hq = q.shape[0]
    g = hq // hk
    out = torch.zeros(hq, d, dtype=F64)
    tol = torch.zeros(hq, d, dtype=F64)
    first = max(0, position - window + 1) if window else 0
    for h in range(hk):
        if position < 0:
            continue
        pages = range(position // page + 1) if listed is None else listed[h]
        rows = [(table[i], t % page) for i in pages for t in range(max(first, i * page), min(position, (i + 1) * page - 1) + 1)
                if 0 <= table[i] < keys.shape[0]]
        if not rows:
            continue
        at, slot = [r[0] for r in rows], [r[1] for r in rows]
        k, v = keys[at, h, slot].to(F64), values[at, h, slot].to(F64)
        for i in range(h * g, (h + 1) * g):
            qi = q[i].to(F64)
            s = k @ qi * scale
            w = torch.softmax(s, 0)
            out[i] = w @ v
            size = w @ v.abs()
            n = len(rows)
            ds = ((d + 8) * 2.0 ** -24 + (2.0 ** -21 if out_type == torch.float32 else 0)) * (k.abs() @ qi.abs()).max() * abs(scale)
            ds = ds + 2.0 ** -22 * s.abs().max()  # the factor of log2(e), the exponent's own rounding
            share = 2 * float(ds) + (n + 64) * 2.0 ** -24 + 2.0 ** -21
            if out_type != torch.float32:
                share += half_step(kept)
                top = float(torch.exp(s - s.max()).sum())
                tol[i] += n * smallest(kept) / top * v.abs().amax(0)
            tol[i] += share * size
    if gate is not None:
        f = torch.sigmoid(gate.to(F64).view(hq, d))
        out, tol = out * f, tol * f + out.abs() * 2.0 ** -21
    return out, tol + half_step(out_type) * out.abs() + smallest(out_type)


def select(q, bounds, table, position, page, count, first=1, last=1, window=0):
    """[kvh][count]: the listed page indexes, then -1; bounds [pages][hk][2][d]."""
    hk = bounds.shape[1]
    g = q.shape[0] // hk
    if position < 0:
        return [[-1] * count for _ in range(hk)]
    begin = (max(0, position - window + 1) if window else 0) // page
    pages = list(range(begin, position // page + 1))
    found = []
    for h in range(hk):
        if len(pages) <= count:
            take = pages
        else:
            score = {}
            for n, i in enumerate(pages):
                if n < first or n >= len(pages) - last:
                    score[i] = math.inf
                    continue
                if not 0 <= table[i] < bounds.shape[0]:
                    score[i] = -math.inf
                    continue
                low, high = bounds[table[i], h].to(F64)
                qh = q[h * g:(h + 1) * g].to(F64)
                score[i] = float(torch.where(qh > 0, qh * high, qh * low).sum().float())  # whatever the bounds hold
            take = sorted(sorted(pages, key=lambda i: (-score[i], i))[:count])
        found.append(take + [-1] * (count - len(take)))
    return found
