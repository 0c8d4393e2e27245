"""Plain 64-bit forms of the operators over long contexts, on the CPU, with the bounds of what the kernels' roundings
may add."""
from __future__ import annotations

import math

import torch

BF16 = torch.finfo(torch.bfloat16).eps / 2   # a rounding to bf16, relative to the value
F32 = 2.0 ** -23                             # a 32-bit operation, however it rounds


def pool(num_pages, page, kv_heads, dim, gen, scale=1.0):
    return (scale * torch.randn((2, num_pages, page, kv_heads, dim), generator=gen)).to(torch.bfloat16)


def tables(lengths, page, gen, *, shared=(), extra=1):
    """Random page tables (-1 behind a sequence's pages) over a pool of the returned size.  ``shared``: per sequence
    (index of the sequence whose first pages it has, number of pages), or nothing."""
    counts = [-(-n // page) for n in lengths]
    have = [s[1] if s else 0 for s in shared] or [0] * len(lengths)
    total = sum(c - h for c, h in zip(counts, have)) + extra
    perm = torch.randperm(total, generator=gen).to(torch.int32)
    t = torch.full((len(lengths), max([1, *counts])), -1, dtype=torch.int32)
    at = 0
    for i, (c, h) in enumerate(zip(counts, have)):
        if h:
            t[i, :h] = t[shared[i][0], :h]
        t[i, h:c] = perm[at:at + c - h]
        at += c - h
    return t, total


def rows(half, table, t0, t1):
    """Tokens [t0, t1) of a sequence from a pool half [NB, BS, Hkv, d], float64 [Hkv, t1 - t0, d]."""
    t = torch.arange(t0, t1)
    page = table.long()[t // half.shape[1]]
    return half[page, t % half.shape[1]].double().transpose(0, 1)


def attend(q, k, v, scale, cap=None, limit=None, scaled_q=False):
    """softmax(scale q k) v of q [n, d], k [t, d], v [t, d] in 64 bits, and the bound of a kernel's error: the weights
    rounded to bf16 once, the output once, logits from 32-bit sums.  ``limit`` [n]: the tokens that each row sees
    (none: a zero row).  ``scaled_q``: q times the scale is rounded to bf16 too, which moves a logit by at most half a
    step of its terms' magnitudes."""
    x = scale * (q @ k.t())
    mag = scale * (q.abs() @ k.abs().t()).max().item() if k.shape[0] else 0.0
    if cap:
        x = cap * torch.tanh(x / cap)
    if limit is not None:
        hidden = torch.arange(k.shape[0]) >= limit[:, None]
        x = x.masked_fill(hidden, -math.inf)
    p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
    out = p @ v
    spread = p @ v.abs()
    # relative, of a weight; twice: of the weight and of the sum
    logit = 2 * ((q.shape[1] + 8) * F32 + (BF16 if scaled_q else 0.0)) * mag + (16 * F32 * cap if cap else 0.0)
    tol = (BF16 * 1.01 + math.expm1(logit) + (32 + k.shape[0] / 16) * F32) * spread + BF16 * out.abs() * 1.02 + 1e-30
    return out, tol


def shared(q, cache, table, lengths, new, scale, cap=None, scaled_q=False):
    """Attention of the last ``new[b]`` tokens of every sequence, rows in order."""
    heads, kv = q.shape[1], cache.shape[3]
    g = heads // kv
    out = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.full(q.shape, 1e-30, dtype=torch.float64)
    at = 0
    for b, n in enumerate(new):
        t = max(0, min(int(lengths[b]), table.shape[1] * cache.shape[2]))
        if n and t:
            safe = table[b].clamp(0, cache.shape[1] - 1)
            k, v = (rows(cache[i], safe, 0, t) for i in (0, 1))
            limit = torch.arange(t - n + 1, t + 1).clamp(min=0).repeat_interleave(g)
            for j in range(kv):
                x = q[at:at + n, j * g:(j + 1) * g].double().reshape(n * g, -1)
                o, e = attend(x, k[j], v[j], scale, cap, limit, scaled_q)
                out[at:at + n, j * g:(j + 1) * g], tol[at:at + n, j * g:(j + 1) * g] = (y.view(n, g, -1) for y in (o, e))
        at += n
    return out, tol


def sparse_decode(q, cache, table, lengths, selected, block, scale, cap=None):
    batch, heads, dim = q.shape
    kv = cache.shape[3]
    g = heads // kv
    out = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.full(q.shape, 1e-30, dtype=torch.float64)
    span = table.shape[1] * cache.shape[2]
    for b in range(batch):
        n = max(0, min(int(lengths[b]), span))
        safe = table[b].clamp(0, cache.shape[1] - 1)
        for j in range(kv):
            pos = [t for c in selected[b, j].tolist() if 0 <= c < -(-n // block)
                   for t in range(c * block, min(n, (c + 1) * block))]
            if not pos:
                continue
            k, v = (rows(cache[i], safe, 0, n)[j][pos] for i in (0, 1))
            s = slice(j * g, (j + 1) * g)
            out[b, s], tol[b, s] = attend(q[b, s].double(), k, v, scale, cap)
    return out, tol


def bounds(cache, table, lengths, new, block, before):
    """The pool of bounds after an update of the last ``new[b]`` tokens."""
    out = before.clone()
    page = cache.shape[2]
    for b, n in enumerate(new):
        t = max(0, min(int(lengths[b]), table.shape[1] * page))
        n = min(n, t)
        if n <= 0:
            continue
        for j in range((t - n) // block, (t - 1) // block + 1):
            p, at = int(table[b, j * block // page]), j * block % page
            if not 0 <= p < cache.shape[1]:
                continue
            k = cache[0, p, at:at + min(block, t - j * block)].double()
            out[p, at // block, :, 0] = k.min(0).values.to(torch.bfloat16)
            out[p, at // block, :, 1] = k.max(0).values.to(torch.bfloat16)
    return out


def scores(q, bnd, table, lengths, page, scale):
    """(scores, bound of the error) in 64 bits; -inf past a sequence's blocks."""
    batch, heads, dim = q.shape
    per, kv = bnd.shape[1], bnd.shape[2]
    g, block = heads // kv, page // per
    out = torch.full((batch, kv, table.shape[1] * per), -math.inf, dtype=torch.float64)
    tol = torch.zeros(out.shape, dtype=torch.float64)
    for b in range(batch):
        n = -(-max(0, min(int(lengths[b]), table.shape[1] * page)) // block)
        for j in range(n):
            x = bnd[int(table[b, j // per].clamp(0, bnd.shape[0] - 1)), j % per].double()   # [Hkv, 2, d]
            y = q[b].double().view(kv, g, 1, dim) * x[:, None]
            out[b, :, j] = scale * y.amax(2).sum(-1).amax(1)
            tol[b, :, j] = scale * y.abs().amax(2).sum(-1).amax(1) * (2 * dim + 4) * F32
    return out, tol


def select(x, lengths, num, block, first, recent):
    out = torch.full((x.shape[0], x.shape[1], num), -1, dtype=torch.int32)
    for b in range(x.shape[0]):
        n = min(-(-max(0, int(lengths[b])) // block), x.shape[2])
        for j in range(x.shape[1]):
            keep = list(range(n))
            if n > num:
                value = [float(y) for y in x[b, j].tolist()]
                value = [-math.inf if math.isnan(y) else y for y in value]
                nan = [math.isnan(float(y)) for y in x[b, j].tolist()]
                middle = sorted(range(first, n - recent), key=lambda i: (nan[i], -value[i], i))
                keep = sorted([*range(first), *middle[:num - first - recent], *range(n - recent, n)])
            out[b, j, :len(keep)] = torch.tensor(keep, dtype=torch.int32)
    return out
