"""Attention over caches in 64 bits, with a bound on what a kernel's result may be off by that follows the data.

Half a step of a type, relative to the value, is eps = torch.finfo(t).eps / 2 (bf16 2^-8, fp16 2^-11).  With
o = sum_j p_j v_j, the terms are, for every row and channel:

  output      eps |o| for the result's own rounding; a rounding that all keys share (equal probabilities, equal values) scales
              o as a whole: eps |o| for the probabilities and eps |o| for the values; half of one is left for what is of second
              order: 3.5 eps |o|.
  p           each probability is rounded to 16 bits on its way into the product with V: sum_j p_j w_j x_j with |x_j| <= eps_p.
              w is |v|, or on a 4-bit cache whatever the probability meets there: the value itself, or its code times the scale,
              with 8 taken off the code or not.  The roundings are independent and have no preferred sign, so by Hoeffding's
              inequality the sum exceeds 8 eps_p sqrt(sum p^2 w^2) with a probability of 2 exp(-32), 3e-14.  A worst-case sum
              (eps_p sum p |v|) is larger than o itself on long caches and would let any result pass.
  v           prompts on a 4-bit cache round the values as well: w is taken sqrt(2) times larger there.
  k           and the keys, independently: the score of key j moves by scale sum_d q_d k_jd y_jd, |y| <= eps_k, which moves o by
              p_j (v_j - o) times that: 8 eps_k sqrt(sum_j p_j^2 s_j^2 (v_j - o)^2), s_j^2 = scale^2 sum_d q_d^2 k_jd^2.
  fp32        a score is a sum of at most eight matrix products whose additions truncate to fp32, 2^-23 of the largest partial sum
              each, below 2^-20 scale sum |q k|; the exponent (scaled to base 2, minus the maximum) and the exponential take
              2^-19.5; the sums of products and their merging 2^-19: p_j is off by less than 2^-18 (1 + scale sum |q k_j| / 4) of
              itself, and all of these may lean one way: 2^-18 sum_j p_j (1 + scale sum |q k_j| / 4) (w_j + |o|).
"""
import math

import torch


def half_step(t):
    return torch.finfo(t).eps / 2


def visible(n, r, window, sinks, device):
    at = torch.arange(n - r, n, device=device)[:, None]
    j = torch.arange(n, device=device)[None, :]
    seen = j <= at
    if window:
        seen &= (j > at - window) | (j < sinks)
    return seen


def clamped(n, r, length, s):
    return min(max(n, 0), length), min(max(r, 0), s)


def attention64(q, k, v, lens, rows, window, sinks, scale, seen_by=visible):
    """The result alone (B, Hq, S, D); rows from rows[b] on hold 7."""
    b, hq, s, d = q.shape
    hkv = k.shape[1]
    out = torch.full((b, hq, s, d), 7.0, dtype=torch.float64, device=q.device)
    for i in range(b):
        n, r = clamped(lens[i], rows[i], k.shape[2], s)
        if r == 0:
            continue
        seen = seen_by(n, r, window, sinks, q.device)
        live = seen.any(0)[:, None]
        kk, vv = (t[i, :, None, :n].double().masked_fill(~live, 0.0) for t in (k, v))
        z = ((q[i, :, :r].double().unflatten(0, (hkv, hq // hkv)) @ kk.transpose(-1, -2)) * scale).masked_fill(~seen, -math.inf)
        out[i, :, :r] = (torch.softmax(z, -1).masked_fill(~seen, 0.0) @ vv).flatten(0, 1)
    return out


def attention_and_bound(q, k, v, lens, rows, window, sinks, scale, dt, eps_p, weight=None, eps_k=0.0):
    """(result, bound), both (B, Hq, S, D); rows from rows[b] on hold 7 and a bound of 0.  `weight`: w above, default |v|."""
    b, hq, s, d = q.shape
    hkv = k.shape[1]
    out = torch.full((b, hq, s, d), 7.0, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    weight = v.abs() if weight is None else weight
    for i in range(b):
        n, r = clamped(lens[i], rows[i], k.shape[2], s)
        if r == 0:
            continue
        seen = visible(n, r, window, sinks, q.device)
        live = seen.any(0)[:, None]
        kk, vv, ww = (t[i, :, None, :n].double().masked_fill(~live, 0.0) for t in (k, v, weight))
        qq = q[i, :, :r].double().unflatten(0, (hkv, hq // hkv))
        z = ((qq @ kk.transpose(-1, -2)) * scale).masked_fill(~seen, -math.inf)
        p = torch.softmax(z, -1).masked_fill(~seen, 0.0)
        o = p @ vv
        e = 3.5 * half_step(dt) * o.abs() + 8 * eps_p * (p.square() @ ww.square()).sqrt()
        if eps_k:
            ps = p.square() * (qq.square() @ kk.square().transpose(-1, -2)) * scale ** 2
            # sum ps (v - o)^2, multiplied out: as a square it cannot be negative
            e += 8 * eps_k * (ps @ vv.square() - 2 * o * (ps @ vv) + o.square() * ps.sum(-1, keepdim=True)).clamp_min(0).sqrt()
        p = p * (1 + (qq.abs() @ kk.abs().transpose(-1, -2)) * (scale / 4))
        e += 2.0 ** -18 * (p @ ww + p.sum(-1, keepdim=True) * o.abs())
        # below the type's smallest normal number its step is constant
        e += half_step(dt) * torch.finfo(dt).smallest_normal * (o != 0)
        out[i, :, :r], bound[i, :, :r] = o.flatten(0, 1), e.flatten(0, 1)
    return out, bound


def worst(got, want, bound):
    """The largest difference as a multiple of the bound (inf: NaN, or a row that has to be exact is not)."""
    diff = (got.double() - want).abs()
    if not torch.isfinite(got.double()).all():
        return math.inf
    at = bound > 0
    if (diff[~at] > 0).any():
        return math.inf
    return float((diff[at] / bound[at]).max()) if at.any() else 0.0


def border_positions(n, r, window, sinks):
    """Positions at which a tile, the window of a row or the first positions begin or end."""
    at = {0, 1, n - r - 1, n - r, n - 1, n // 2} | {m for t in (16, 64, 128) for m in (t - 1, t, n // t * t - 1, n // t * t)}
    if window:
        at |= {sinks - 1, sinks} | {x - window + e for x in (n - r, n - 1) for e in (0, 1, 2)}
    return sorted(x for x in at if 0 <= x < n)


def marked(x, lens, rows, window, sinks, factor=16.0):
    """The rows x (B, H, L, D) with those at borders made larger, so that one of them lost or gained shows."""
    x = x.clone()
    for i in range(x.shape[0]):
        n, r = clamped(lens[i], rows[i], x.shape[2], 1 << 30)
        x[i, :, border_positions(n, r, window, sinks)] *= factor
    return x


def quantise64(x):
    """Codes (as whole numbers), s and lo of rows x (..., D) of a 16-bit type, quotients in 64 bits."""
    g = x.unflatten(-1, (-1, 64))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi.float() - lo.float()) / torch.full_like(hi, 15, dtype=torch.float32)).to(x.dtype)    # (a scalar divisor would become a factor 1/15)
    c = torch.where(s > 0, ((g.double() - lo.double()) / s.double()).round().clamp(0, 15), torch.zeros((), dtype=torch.float64, device=x.device))
    return c.flatten(-2), s.squeeze(-1), lo.squeeze(-1)


def values64(codes, meta):
    """What packed codes (..., D / 2) and meta (..., D / 64, 2) stand for, and the weight w of a probability on them."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, 64)).double()
    s = meta[..., :1].double()
    x = meta[..., 1:].double() + c * s
    return x.flatten(-2), torch.maximum(x.abs(), s * torch.maximum(c, (c - 8).abs())).flatten(-2)


def pack4(c):
    c = c.to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4)
