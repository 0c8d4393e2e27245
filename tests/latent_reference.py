"""Latent attention and the rotation in float64, with the spread that the kernels' bf16 roundings leave.

Every rounding to bf16 moves a value x by at most u |x|, u = 2^-8, to either side.  The kernels round several
quantities that then enter sums, so the error of an output is a weighted sum of independent errors of that size; a
uniform error on [-a, a] is sub-Gaussian with variance proxy a^2 / 3, so a sum with proxy s^2 passes 6 s with
probability below 2 exp(-18) = 3e-8.  ``attend`` returns s next to the output.  Its terms, for weights p_j, values
v_j, result o (all per head):

  absorbed form: softmax weights    sum_j (p_j v_j)^2
                 absorbed q         sum_r (q_r scale sum_j p_j c_jr (v_j - o))^2
                 latent-wide result sum_r (o_r W_uv,r)^2
  expanded form: softmax weights    sum_j (p_j v_j)^2
                 expanded keys      sum_j (p_j (v_j - o) scale)^2 sum_d (q_d k_jd)^2
                 expanded values    sum_j (p_j v_j)^2
  both:          the output         o^2

each times u^2 / 3."""
from __future__ import annotations

import math

import torch

U = 2.0 ** -8


def attend(q_nope, q_rope, rows, w_uk, w_uv, seen, scale, form):
    """One sequence and head: q_nope [n, Dn], q_rope [n, Dr], rows [L, R + Dr], w_uk [Dn, R], w_uv [Dv, R]; row i
    sees the first seen[i] cache rows.  Returns (out, spread), float64 [n, Dv]."""
    qn, qr, rows, w_uk, w_uv = (t.double() for t in (q_nope, q_rope, rows, w_uk, w_uv))
    r = w_uk.shape[1]
    n, dv = qn.shape[0], w_uv.shape[0]
    out = torch.zeros((n, dv), dtype=torch.float64, device=qn.device)
    spread = torch.zeros_like(out)
    for i in range(n):
        m = int(seen[i])
        if m <= 0:
            continue
        c, kr = rows[:m, :r], rows[:m, r:]
        k, v = c @ w_uk.t(), c @ w_uv.t()
        p = torch.softmax((k @ qn[i] + kr @ qr[i]) * scale, 0)
        o = p @ v
        var = ((p[:, None] * v) ** 2).sum(0) + o ** 2
        d = v - o
        if form == "absorbed":
            q_lat, o_lat = qn[i] @ w_uk, p @ c
            m_rd = (p[:, None] * c).t() @ d
            var = var + ((q_lat * scale)[:, None] * m_rd).square().sum(0) + (w_uv * o_lat).square().sum(1)
        else:
            ks = ((qn[i] * k) ** 2).sum(1)
            var = var + ((p[:, None] * d * scale) ** 2 * ks[:, None]).sum(0) + ((p[:, None] * v) ** 2).sum(0)
        out[i], spread[i] = o, torch.sqrt(var / 3) * U
    return out, spread


def check(got, want, spread, what=""):
    """|got - want| <= 6 s, and 2^-18 of the largest value for the float32 sums."""
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    err = (got - want).abs()
    bound = 6 * spread + 2.0 ** -18 * want.abs().max()
    worst = float((err - bound).max())
    ratio = float((err / bound.clamp_min(1e-30)).max())
    print(f"{what}: max-abs err {float(err.max()):.3e}, {ratio:.2f} of the bound", flush=True)
    assert worst <= 0, f"{what}: error passes its bound by {worst:.3e}"


def angles(positions, freq):
    return positions.double()[:, None] * freq.double()[None, :]


def rotate(x, positions, freq, amp, interleaved):
    """x [T, H, r] in float64."""
    x = x.double()
    a = angles(positions, freq)[:, None]
    c, s = torch.cos(a) * amp, torch.sin(a) * amp
    r = x.shape[-1]
    p, q = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :r // 2], x[..., r // 2:])
    y = (p * c - q * s, p * s + q * c)
    size = (p.abs() + q.abs()) * amp
    if interleaved:
        return torch.stack(y, -1).flatten(-2), torch.stack((size, size), -1).flatten(-2)
    return torch.cat(y, -1), torch.cat((size, size), -1)


def yarn_frequencies(r, base, factor, span, fast=32.0, slow=1.0):
    """Pair by pair, from the definition."""
    low = max(math.floor(r * math.log(span / (fast * 2 * math.pi)) / (2 * math.log(base))), 0)
    high = min(math.ceil(r * math.log(span / (slow * 2 * math.pi)) / (2 * math.log(base))), r - 1)
    out = []
    for i in range(r // 2):
        f = base ** (-2 * i / r)
        t = min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0)
        out.append(f / factor * t + f * (1 - t))
    return out
