"""The 4-bit KV cache (append, read, attention) and windowed attention over 16-bit caches against plain 64-bit forms.

Tolerances.  eps is half a step of the type relative to the value (bf16 2^-8, fp16 2^-11: torch.finfo(t).eps / 2 is what
one rounding is off by at most).  Reading back is one rounding of lo + c s: |lo| and |c s| may cancel, but the fused
multiply-add rounds their exact sum once, so the bound is half a step of the result.  Attention: the output's own rounding
is half a step of |o|.  Besides, every probability and (4-bit values, or a cache read back for a prompt) every key and
value may be rounded to the 16-bit type on its way into a matrix product.  A rounded probability changes o by at most
half a step of sum p |v| <= max |v|, a rounded value by half a step of max |v|; rounded keys change a score by at most
half a step of scale * sum |q k|, hence every probability by that much relative, hence o by at most twice that times
max |v| (the tests allow no more than four half steps for it).  The tests' bound is the sum of these.
"""
import math

import pytest
import torch

from trinity_b200 import _lib as L
from trinity_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16]


def half_step(t):
    return torch.finfo(t).eps / 2


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def quantise64(x):
    """Codes and (s, lo) of rows x (..., D), quotients in 64 bits."""
    g = x.unflatten(-1, (-1, 64))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi.float() - lo.float()) / torch.full_like(hi, 15, dtype=torch.float32)).to(x.dtype)    # (a scalar divisor would become a factor 1/15)
    c = torch.where(s > 0, ((g.double() - lo.double()) / s.double()).round().clamp(0, 15), torch.zeros((), dtype=torch.float64, device=x.device))
    return c.flatten(-2), s.squeeze(-1), lo.squeeze(-1)


def values64(cache, which):
    codes, meta = (cache.k_codes, cache.k_meta) if which == "k" else (cache.v_codes, cache.v_meta)
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, 64)).double()
    return (meta[..., 1:].double() + c * meta[..., :1].double()).flatten(-2)


def filled_cache(b, h, length, d, dt, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    cache = ops.kv4_cache(b, h, length, d, dt, DEV)
    k = torch.randn(b, h, length, d, generator=g, device=DEV) * scale + torch.randn(1, h, 1, d, generator=g, device=DEV)
    v = torch.randn(b, h, length, d, generator=g, device=DEV) * scale
    for x, codes, meta in ((k, cache.k_codes, cache.k_meta), (v, cache.v_codes, cache.v_meta)):
        c, s, lo = quantise64(x.to(dt))
        c = c.to(torch.uint8)
        codes[:, :, :length] = c[..., 0::2] | (c[..., 1::2] << 4)
        meta[:, :, :length] = torch.stack([s, lo], -1)
    return cache


def visible(n, r, window, sinks):
    at = torch.arange(n - r, n, device=DEV)[:, None]
    j = torch.arange(n, device=DEV)[None, :]
    seen = j <= at
    if window:
        seen &= (j > at - window) | (j < sinks)
    return seen


def attention64(q, k, v, lens, rows, window, sinks, scale):
    """(out, bound-making sums) of every row; q (B,Hq,S,D), k, v (B,Hkv,L,D) in 64 bits; rows past rows[b] stay NaN."""
    b, hq, s, d = q.shape
    hkv, length = k.shape[1], k.shape[2]
    out = torch.full((b, hq, s, d), math.nan, dtype=torch.float64, device=DEV)
    q = q.double().unflatten(1, (hkv, hq // hkv))
    for i in range(b):
        n, r = min(max(lens[i], 0), length), min(max(rows[i], 0), s)
        if r == 0:
            continue
        seen = visible(n, r, window, sinks)
        z = (q[i, :, :, :r] @ k[i, :, None, :n].transpose(-1, -2)) * scale
        z = z.masked_fill(~seen, -math.inf)
        p = torch.softmax(z, -1).masked_fill(~seen, 0.0)    # a row that sees nothing: zeros
        out[i, :, :r] = (p @ v[i, :, None, :n].masked_fill(~seen.any(0)[:, None], 0.0)).flatten(0, 1)
    return out


def check_rows(got, want, q, k, v, lens, rows, scale, dt):
    """Rows below rows[b] within the bound derived above; the others untouched (they held 7)."""
    eps = half_step(dt)
    for i in range(q.shape[0]):
        n, r = min(max(lens[i], 0), k.shape[2]), min(max(rows[i], 0), q.shape[2])
        assert torch.equal(got[i, :, r:], torch.full_like(got[i, :, r:], 7.0)), "rows behind the sequence were written"
        if r == 0:
            continue
        g, w = got[i, :, :r].double(), want[i, :, :r]
        assert torch.isfinite(g).all()
        if n == 0:
            assert torch.equal(g, torch.zeros_like(g))
            continue
        vmax = v[i, :, :n].abs().amax()
        score = scale * (q[i].double().abs().amax((0, 1)) * k[i, :, :n].abs().amax((0, 1))).sum()
        bound = eps * (w.abs() + vmax * (2 + min(2 * score, 4.0)))
        assert ((g - w).abs() <= bound).all(), f"sequence {i}: {float(((g - w).abs() / bound).max()):.2f} times the bound"


# ------------------------------------------------------------------------------------------------ append and read
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("b,h,s,d,length", [(1, 1, 1, 64, 4), (2, 3, 1, 128, 32), (3, 2, 77, 128, 200), (2, 8, 257, 64, 512), (1, 71, 5, 64, 8)])
def test_append_codes_and_meta(dt, b, h, s, d, length):
    g = torch.Generator(device=DEV).manual_seed(s)
    cache = ops.Kv4Cache(*[t.fill_(9) for t in ops.kv4_cache(b, h, length, d, dt, DEV)])
    before = [t.clone() for t in cache]
    k = torch.randn(b, s, h, d, generator=g, device=DEV).to(dt).transpose(1, 2)      # a projection's layout
    v = (torch.randn(b, h, s, d, generator=g, device=DEV) * 30).to(dt)
    start = [max(0, (length - s) // (i + 1)) for i in range(b)]
    rows = [max(1, s - 3 * i) for i in range(b)]
    ops.kv4_append(cache, k, v, ints(start), rows=ints(rows))
    for x, codes, meta, c0, m0 in ((k, cache.k_codes, cache.k_meta, before[0], before[2]), (v, cache.v_codes, cache.v_meta, before[1], before[3])):
        c, sc, lo = quantise64(x)
        for i in range(b):
            a, e = start[i], start[i] + rows[i]
            got = torch.stack([codes[i] & 15, codes[i] >> 4], -1).flatten(-2)[:, a:e].double()
            assert torch.equal(got, c[i, :, :rows[i]])
            assert torch.equal(meta[i, :, a:e, :, 0], sc[i, :, :rows[i]]) and torch.equal(meta[i, :, a:e, :, 1], lo[i, :, :rows[i]])
            keep = torch.ones(length, dtype=torch.bool, device=DEV)
            keep[a:e] = False
            assert torch.equal(codes[i][:, keep], c0[i][:, keep]) and torch.equal(meta[i][:, keep], m0[i][:, keep])


@pytest.mark.parametrize("dt", TYPES)
def test_append_borders_and_odd_groups(dt):
    """Quotients on and next to borders, equal values, subnormal steps, infinities and NaN."""
    tiny = torch.finfo(dt).smallest_normal
    rows = [torch.arange(64) % 16, torch.arange(64) % 31 / 2.0, torch.full((64,), 3.25), torch.arange(64) % 16 * tiny / 64, torch.arange(64) * 0.0]
    rows += [(torch.arange(64) % 31) * (2.0 ** e) * 0.3 for e in (-6, 0, 5)]
    rows += [torch.linspace(-1, 1, 64) * 37.3 + o for o in (0.0, 512.0, -0.01)]
    top = torch.finfo(dt).max
    rows += [torch.tensor([top, -top] * 32) / (1.0 if dt == torch.float16 else 4.0)]
    x = torch.stack([r.double() for r in rows]).to(dt).to(DEV)[None, None]                # (1, 1, rows, 64)
    bad = torch.ones(3, 64, dtype=dt, device=DEV)
    bad[0, 5], bad[1, 63], bad[2, 0] = math.inf, math.nan, -math.inf
    both = torch.cat([x, bad[None, None]], 2)
    cache = ops.kv4_cache(1, 1, both.shape[2], 64, dt, DEV)
    ops.kv4_append(cache, both, both, 0)
    c, s, lo = quantise64(x)
    n = x.shape[2]
    got = torch.stack([cache.k_codes & 15, cache.k_codes >> 4], -1).flatten(-2)[:, :, :n].double()
    assert torch.equal(got, c) and torch.equal(cache.k_meta[:, :, :n, :, 0], s) and torch.equal(cache.k_meta[:, :, :n, :, 1], lo)
    k, v = ops.kv4_read(cache, 0, both.shape[2])
    assert torch.isnan(k[:, :, n:]).all() and torch.isnan(v[:, :, n:]).all() and torch.isfinite(k[:, :, :n]).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("b,h,count,d,length", [(1, 1, 1, 64, 4), (2, 2, 33, 128, 64), (3, 8, 130, 64, 300), (2, 4, 64, 128, 64)])
def test_read(dt, b, h, count, d, length):
    cache = filled_cache(b, h, length, d, dt, 3)
    start = [(length - count) // (i + 1) for i in range(b)]
    rows = [count - i for i in range(b)]
    k = torch.full((b, count, h, d), 7.0, dtype=dt, device=DEV).transpose(1, 2)
    v = torch.full((b, h, count, d), 7.0, dtype=dt, device=DEV)
    ops.kv4_read(cache, ints(start), count, rows=ints(rows), k_out=k, v_out=v)
    for out, which in ((k, "k"), (v, "v")):
        want = values64(cache, which)
        for i in range(b):
            w = want[i, :, start[i]:start[i] + rows[i]]
            # one rounding of the exact sum; below the type's smallest normal number its step is constant
            assert ((out[i, :, :rows[i]].double() - w).abs() <= half_step(dt) * w.abs().clamp_min(torch.finfo(dt).smallest_normal)).all()
            assert torch.equal(out[i, :, rows[i]:], torch.full_like(out[i, :, rows[i]:], 7.0))


def test_positions_outside_the_cache_are_skipped():
    dt = torch.bfloat16
    cache = filled_cache(2, 2, 16, 64, dt, 5)
    before = [t.clone() for t in cache]
    x = torch.randn(2, 2, 6, 64, device=DEV).to(dt)
    ops.kv4_append(cache, x, x, ints([13, -2]))
    c, s, lo = quantise64(x)
    got = torch.stack([cache.k_codes & 15, cache.k_codes >> 4], -1).flatten(-2).double()
    assert torch.equal(got[0, :, 13:], c[0, :, :3]) and torch.equal(got[1, :, :4], c[1, :, 2:])
    assert torch.equal(cache.v_codes[0, :, :13], before[1][0, :, :13]) and torch.equal(cache.v_codes[1, :, 4:], before[1][1, :, 4:])
    k, v = ops.kv4_read(cache, ints([14, -3]), 5)
    assert torch.equal(k[0, :, 2:], torch.zeros_like(k[0, :, 2:])) and torch.equal(k[1, :, :3], torch.zeros_like(k[1, :, :3]))
    for rows in ([0, 0], [-4, -1]):
        keep = [t.clone() for t in cache]
        ops.kv4_append(cache, x, x, 0, rows=ints(rows))
        assert all(torch.equal(a, b) for a, b in zip(keep, cache))


# ------------------------------------------------------------------------------------------------ attention
SHAPES = [  # b, hq, hkv, d, s, cache length, lens, rows, window, sinks
    (1, 1, 1, 64, 1, 4, [1], [1], 0, 0),
    (1, 8, 2, 128, 1, 1040, [1037], [1], 0, 0),
    (3, 8, 8, 128, 1, 300, [300, 1, 129], [1, 1, 1], 0, 0),
    (2, 71, 1, 64, 1, 512, [511, 257], [1, 1], 0, 0),
    (4, 16, 4, 64, 1, 2048, [2048, 0, 1000, 31], [1, 1, 0, 1], 0, 0),
    (2, 14, 2, 128, 1, 4096, [4001, 333], [1, 1], 128, 4),
    (2, 4, 4, 64, 3, 640, [640, 2], [3, 3], 33, 1),
    (3, 32, 8, 128, 5, 1000, [999, 400, 64], [5, 2, 4], 200, 16),
    (2, 32, 8, 128, 7, 512, [512, 100], [7, 7], 0, 0),
    (2, 8, 1, 128, 17, 300, [290, 17], [17, 11], 0, 0),
    (1, 4, 2, 128, 130, 132, [130], [130], 0, 0),
    (2, 8, 2, 128, 300, 700, [700, 299], [300, 299], 0, 0),
    (2, 8, 2, 64, 257, 1024, [1021, 600], [257, 100], 100, 4),
    (3, 4, 4, 128, 140, 900, [888, 100, 0], [140, 140, 140], 65, 33),
    (2, 6, 2, 64, 513, 516, [514, 513], [513, 400], 1, 0),
    (2, 6, 2, 128, 260, 1200, [1111, 300], [260, 260], 128, 300),
    (1, 2, 1, 128, 40, 20000, [19999], [40], 5000, 128),
    (2, 14, 2, 64, 45, 400, [400, 45], [45, 30], 50, 3),
    (1, 71, 1, 64, 40, 300, [300], [39], 0, 0),
    (2, 12, 2, 128, 100, 1000, [900, 100], [100, 64], 150, 20),
    (3, 32, 8, 128, 300, 2048, [2000, 300, 20], [300, 290, 300], 700, 4),
    (2, 16, 2, 64, 33, 3000, [3000, 1029], [33, 32], 0, 0),
    (2, 8, 2, 128, 1, 30000, [30000, 777], [1, 1], 0, 0),
    (3, 12, 2, 64, 2, 40000, [40000, 9, 20011], [2, 1, 2], 0, 0),
    (2, 20, 2, 128, 1, 24000, [11, 23999], [1, 1], 12000, 100),
    (70, 16, 8, 64, 1, 600, [600 - 8 * i for i in range(70)], [1] * 69 + [0], 0, 0),
    (40, 8, 8, 128, 2, 400, [10 * i for i in range(40)], [2] * 40, 0, 0),
    (33, 4, 2, 64, 300, 400, [i * 12 for i in range(33)], [(i * 97) % 301 for i in range(33)], 0, 0),
    (128, 2, 2, 128, 270, 320, [320 - i for i in range(128)], [0] * 127 + [270], 50, 4),
    (129, 2, 1, 64, 90, 128, [i % 129 for i in range(129)], [i % 91 for i in range(129)], 0, 0),
    (3, 4, 2, 64, 80, 4000, [4000, 2222, 0], [80, 0, 33], 0, 0),
    (2, 71, 1, 64, 1, 60000, [60000, 12345], [1, 1], 0, 0),
    (9, 96, 4, 64, 2, 2100, [i * 240 for i in range(9)], [2, 1, 0] * 3, 0, 0),
    (38, 192, 8, 64, 1, 200, [200 - 5 * i for i in range(38)], [1] * 38, 64, 2),
]


def case(shape, dt, seed=11):
    b, hq, hkv, d, s, length, lens, rows, window, sinks = shape
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(b, s, hq, d, generator=g, device=DEV).to(dt).transpose(1, 2)
    out = torch.full((b, s, hq, d), 7.0, dtype=dt, device=DEV).transpose(1, 2)
    return q, out, dict(window=window, sinks=sinks, sm_scale=d ** -0.5, q_rows=ints(rows), out=out)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_kv4_attn(shape, dt):
    b, hq, hkv, d, s, length, lens, rows, window, sinks = shape
    cache = filled_cache(b, hkv, length, d, dt, 7)
    q, out, kw = case(shape, dt)
    ops.kv4_attn(q, cache, ints(lens), **kw)
    ops.device_status()
    k, v = values64(cache, "k"), values64(cache, "v")
    want = attention64(q, k, v, lens, rows, window, sinks, d ** -0.5)
    check_rows(out, want, q, k, v, lens, rows, d ** -0.5, dt)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attn_window(shape, dt):
    b, hq, hkv, d, s, length, lens, rows, window, sinks = shape
    g = torch.Generator(device=DEV).manual_seed(7)
    k = (torch.randn(b, hkv, length, d, generator=g, device=DEV) + torch.randn(1, hkv, 1, d, generator=g, device=DEV)).to(dt)
    v = torch.randn(b, length, hkv, d, generator=g, device=DEV).to(dt).transpose(1, 2)    # another order of axes
    q, out, kw = case(shape, dt)
    ops.attn_window(q, k, v, ints(lens), **kw)
    ops.device_status()
    want = attention64(q, k.double(), v.double(), lens, rows, window, sinks, d ** -0.5)
    check_rows(out, want, q, k.double(), v.double(), lens, rows, d ** -0.5, dt)


@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("size,flat", [(1e30, True), (1e30, False), (3e7, True), (1.0, True), (1e-5, False), (1e-12, False), (1e-12, True)])
def test_kv4_attn_values_of_any_size(size, flat, rows):
    """V scales and minima far from 1, or no scale at all (a group of equal values); keys whose scale is 0."""
    dt, b, hq, hkv, d, length, n = torch.bfloat16, 1, 4, 1, 128, 512, 500
    cache = filled_cache(b, hkv, length, d, dt, 7)
    g = torch.Generator(device=DEV).manual_seed(2)
    v = torch.randn(b, hkv, length, 2 if flat else d, generator=g, device=DEV).repeat_interleave(64 if flat else 1, -1) * size
    k = torch.randn(b, hkv, length, 2, generator=g, device=DEV).repeat_interleave(64, -1)
    ops.kv4_append(cache, k.to(dt), v.to(dt), 0)
    q = torch.randn(b, hq, rows, d, generator=g, device=DEV).to(dt)
    out = torch.full((b, hq, rows, d), 7.0, dtype=dt, device=DEV)
    ops.kv4_attn(q, cache, ints([n]), sm_scale=0.1, out=out)
    k64, v64 = values64(cache, "k"), values64(cache, "v")
    check_rows(out, attention64(q, k64, v64, [n], [rows], 0, 0, 0.1), q, k64, v64, [n], [rows], 0.1, dt)


@pytest.mark.parametrize("s", [1, 4, 130])
@pytest.mark.parametrize("kv4", [True, False])
def test_rows_nobody_sees_may_hold_anything(kv4, s):
    """NaN and infinities behind the sequence and between the first positions and the window: same bits as with zeros there."""
    dt, b, hq, hkv, d, length, n, window, sinks = torch.bfloat16, 1, 4, 2, 128, 1024, 900, 130, 5
    q = torch.randn(b, hq, s, d, device=DEV).to(dt)
    hidden = torch.ones(length, dtype=torch.bool, device=DEV)
    hidden[:sinks] = False
    hidden[n - s - window + 1:n] = False
    outs = []
    for fill in (0.0, math.nan, math.inf):
        if kv4:
            cache = filled_cache(b, hkv, length, d, dt, 7)
            for t in (cache.k_meta, cache.v_meta):
                t[:, :, hidden] = fill
            outs.append(ops.kv4_attn(q, cache, ints([n]), window=window, sinks=sinks, sm_scale=0.1))
        else:
            g = torch.Generator(device=DEV).manual_seed(3)
            k, v = (torch.randn(b, hkv, length, d, generator=g, device=DEV).to(dt) for _ in range(2))
            k[:, :, hidden], v[:, :, hidden] = fill, fill
            outs.append(ops.attn_window(q, k, v, ints([n]), window=window, sinks=sinks, sm_scale=0.1))
    assert torch.isfinite(outs[0]).all() and torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("length", [2048, 24000])
@pytest.mark.parametrize("kv4", [True, False])
def test_same_bits_every_time_and_from_a_graph(kv4, length):
    shape = (5, 16, 4, 128, 1, length, [length, 77, 1500, 0, 640], [1] * 5, 0, 0)
    b, hq, hkv, d, s, length, lens, rows, window, sinks = shape
    dt = torch.float16
    q, out, kw = case(shape, dt)
    lens = ints(lens)
    if kv4:
        cache = filled_cache(b, hkv, length, d, dt, 7)
        call = lambda: ops.kv4_attn(q, cache, lens, **kw)
    else:
        k, v = (torch.randn(b, hkv, length, d, device=DEV).to(dt) for _ in range(2))
        call = lambda: ops.attn_window(q, k, v, lens, **kw)
    call()
    first = out.clone()
    out.fill_(7)
    call()
    assert torch.equal(out, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    lens.copy_(ints([1, 2000, 64, 333, 65]))     # the lengths are read on the device
    graph.replay()
    replayed = out.clone()
    out.fill_(7)
    call()
    assert torch.equal(out, replayed) and not torch.equal(out, first)


def test_write_then_attend_token_by_token():
    """As a server runs them: a ragged batch of prompts is written and attended to, then token after token."""
    dt, b, hq, hkv, d, length = torch.bfloat16, 3, 8, 2, 128, 256
    scale, window, sinks = d ** -0.5, 60, 4
    g = torch.Generator(device=DEV).manual_seed(1)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dt)
    prompts = [100, 7, 64]
    cache = ops.kv4_cache(b, hkv, length, d, dt, DEV)
    held = torch.zeros(b, hkv, length, d, dtype=dt, device=DEV)          # what the 4-bit cache stands for, in 16 bits
    held_v = torch.zeros_like(held)
    lens = [0] * b
    for new in [prompts] + [[1, 1, 1]] * 4 + [[3, 0, 2]]:
        s = max(new)
        q, k, v = rn(b, s, hq, d).transpose(1, 2), rn(b, s, hkv, d).transpose(1, 2), rn(b, s, hkv, d).transpose(1, 2)
        start, rows = ints(lens), ints(new)
        ops.kv4_append(cache, k, v, start, rows=rows)
        lens = [x + y for x, y in zip(lens, new)]
        out = torch.full((b, s, hq, d), 7.0, dtype=dt, device=DEV).transpose(1, 2)
        ops.kv4_attn(q, cache, ints(lens), window=window, sinks=sinks, sm_scale=scale, q_rows=rows, out=out)
        k64, v64 = values64(cache, "k"), values64(cache, "v")
        check_rows(out, attention64(q, k64, v64, lens, new, window, sinks, scale), q, k64, v64, lens, new, scale, dt)
        kr, vr = ops.kv4_read(cache, start, s, rows=rows)
        for i in range(b):
            held[i, :, lens[i] - new[i]:lens[i]], held_v[i, :, lens[i] - new[i]:lens[i]] = kr[i, :, :new[i]], vr[i, :, :new[i]]
        out16 = torch.full((b, s, hq, d), 7.0, dtype=dt, device=DEV).transpose(1, 2)
        ops.attn_window(q, held, held_v, ints(lens), window=window, sinks=sinks, sm_scale=scale, q_rows=rows, out=out16)
        check_rows(out16, attention64(q, held.double(), held_v.double(), lens, new, window, sinks, scale), q, held.double(), held_v.double(),
                   lens, new, scale, dt)
    assert ops.device_status() == 0


def test_empty_batches_and_no_rows():
    dt = torch.bfloat16
    for b, s in ((0, 3), (2, 0)):
        cache = ops.kv4_cache(b, 2, 16, 64, dt, DEV)
        x = torch.zeros(b, 2, s, 64, dtype=dt, device=DEV)
        lens = torch.zeros(b, dtype=torch.int32, device=DEV)
        ops.kv4_append(cache, x, x, 0)
        assert ops.kv4_read(cache, 0, s)[0].shape == (b, 2, s, 64)
        assert ops.kv4_attn(x, cache, lens).shape == (b, 2, s, 64)
        assert ops.attn_window(x, torch.zeros(b, 2, 16, 64, dtype=dt, device=DEV), torch.zeros(b, 2, 16, 64, dtype=dt, device=DEV), lens, window=4).shape == x.shape


def test_offsets_past_32_bits():
    """Caches whose codes, or whose 16-bit rows, take more than 4 GiB: rows at the far end, and a window there."""
    dt, d, h = torch.bfloat16, 128, 2
    g = torch.Generator(device=DEV).manual_seed(4)
    for kv4, length in ((True, 40_000_000), (False, 12_000_000)):
        new, window, sinks = 20, 100, 4
        n = length - 8
        q, k, v = (torch.randn(1, x, new, d, generator=g, device=DEV).to(dt) for x in (4, h, h))
        first, tail = slice(0, sinks), slice(n - new - window, n)
        if kv4:
            cache = ops.Kv4Cache(*[torch.empty(1, h, length, d // 2, dtype=torch.uint8, device=DEV) for _ in range(2)],
                                 *[torch.empty(1, h, length, d // 64, 2, dtype=dt, device=DEV) for _ in range(2)])
            old = torch.randn(1, h, window, d, generator=g, device=DEV).to(dt)
            ops.kv4_append(cache, old, old, 0, rows=ints([sinks]))
            ops.kv4_append(cache, old, old, n - new - window)
            ops.kv4_append(cache, k, v, n - new)
            kr, vr = ops.kv4_read(cache, n - new, new)
            assert ((kr.double() - k.double()).abs() <= (k.double().amax(-1) - k.double().amin(-1)).amax() / 15).all()
            outs = [ops.kv4_attn(q[:, :, -r:], cache, ints([n]), window=window, sinks=sinks, sm_scale=0.1) for r in (1, new)]
            part = ops.Kv4Cache(*[torch.cat([t[:, :, first], t[:, :, tail]], 2).contiguous() for t in cache])
            k64, v64 = values64(part, "k"), values64(part, "v")
        else:
            kc, vc = torch.empty(1, h, length, d, dtype=dt, device=DEV), torch.empty(1, h, length, d, dtype=dt, device=DEV)
            for t, x in ((kc, k), (vc, v)):
                t[:, :, first] = torch.randn(1, h, sinks, d, generator=g, device=DEV).to(dt)
                t[:, :, tail] = torch.randn(1, h, window + new, d, generator=g, device=DEV).to(dt)
                t[:, :, n - new:n] = x
            outs = [ops.attn_window(q[:, :, -r:], kc, vc, ints([n]), window=window, sinks=sinks, sm_scale=0.1) for r in (1, new)]
            k64, v64 = (torch.cat([t[:, :, first], t[:, :, tail]], 2).double() for t in (kc, vc))
            del kc, vc
        # the same keys in a short cache, with the window at the same distance: the first ones stay, the rest is the tail
        m = sinks + window + new
        for r, out in zip((1, new), outs):
            at = torch.arange(m - r, m, device=DEV)[:, None]
            j = torch.arange(m, device=DEV)[None, :]
            seen = (j <= at) & ((j > at - window) | (j < sinks))
            z = torch.einsum("bhgrd,bhnd->bhgrn", q[:, :, -r:].double().unflatten(1, (h, 2)), k64) * 0.1
            p = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
            want = torch.einsum("bhgrn,bhnd->bhgrd", p, v64).flatten(1, 2)
            check_rows(out, want, q[:, :, -r:], k64, v64, [m], [r], 0.1, dt)
        del outs


def test_two_streams_at_once():
    """Calls on two streams have workspaces of their own."""
    shape = (4, 32, 8, 128, 1, 24000, [24000, 4000, 100, 9999], [1] * 4, 0, 0)
    b, hq, hkv, d, s, length, lens, rows, window, sinks = shape
    caches = [filled_cache(b, hkv, length, d, torch.bfloat16, i) for i in range(2)]
    q, _, kw = case(shape, torch.bfloat16)
    del kw["out"]
    want = [ops.kv4_attn(q, c, ints(lens), **kw).clone() for c in caches]
    lens = ints(lens)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            got.append([ops.kv4_attn(q, caches[i], lens, **kw) for _ in range(20)])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("kv4", [True, False])
def test_two_captured_graphs_at_once(kv4, new):
    """Graphs captured one after the other on one stream have workspaces of their own, and none with eager calls."""
    shape = (4, 32, 8, 128, new, 24000, [24000, 4000, 100, 9999], [new] * 4, 0, 0)
    b, hq, hkv, d, s, length, lens, rows, window, sinks = shape
    lens = ints(lens)
    q, _, kw = case(shape, torch.bfloat16)
    del kw["out"]
    g = torch.Generator(device=DEV).manual_seed(3)
    if kv4:
        caches = [filled_cache(b, hkv, length, d, torch.bfloat16, i) for i in range(3)]
        calls = [lambda c=c: ops.kv4_attn(q, c, lens, **kw) for c in caches]
    else:
        caches = [torch.randn(b, hkv, length, d, generator=g, device=DEV).bfloat16() for _ in range(3)]
        calls = [lambda c=c: ops.attn_window(q, c, c, lens, **kw) for c in caches]
    want = [f().clone() for f in calls]
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph, f in zip(graphs, calls):
        with torch.cuda.graph(graph):
            outs.append(f())
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        eager = calls[2]()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[2])


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals_on_the_device():
    dt = torch.bfloat16
    cache = filled_cache(2, 2, 16, 64, dt, 5)
    x = torch.zeros(2, 2, 3, 64, dtype=dt, device=DEV)
    lens = ints([3, 3])
    q = torch.zeros(2, 4, 3, 64, dtype=dt, device=DEV)
    with pytest.raises(TypeError):
        ops.kv4_append(cache, x.half(), x.half(), 0)
    with pytest.raises(ValueError):
        ops.kv4_append(cache, x[:, :1], x[:, :1], 0)
    with pytest.raises(ValueError):
        ops.kv4_append(cache, torch.zeros(2, 2, 64, 3, dtype=dt, device=DEV).transpose(2, 3), x, 0)
    with pytest.raises(L.Tb200Error):       # a row step that is no multiple of 16 bytes
        ops.kv4_append(cache, torch.zeros(2, 2, 3, 68, dtype=dt, device=DEV)[..., :64], x, 0)
    with pytest.raises(TypeError):
        ops.kv4_append(cache, x, x, torch.zeros(2, dtype=torch.int64, device=DEV))
    for bad in (None, 1.5, [0, 0]):
        with pytest.raises(TypeError):
            ops.kv4_append(cache, x, x, bad)
        with pytest.raises(TypeError):
            ops.kv4_attn(q, cache, bad)
    with pytest.raises(ValueError):
        ops.kv4_append(cache, x, x, 1 << 40)
    with pytest.raises(L.Tb200Error):       # both results in one place
        ops.kv4_read(cache, 0, 3, k_out=x, v_out=x)
    with pytest.raises(L.Tb200Error):       # written rows that overlap
        ops.kv4_read(cache, 0, 3, k_out=torch.zeros(1, 2, 3, 64, dtype=dt, device=DEV).expand(2, 2, 3, 64), v_out=x.clone())
    with pytest.raises(ValueError):
        ops.kv4_attn(q.cpu(), cache, lens)
    with pytest.raises(ValueError):
        ops.kv4_attn(q, ops.Kv4Cache(cache.k_codes, cache.v_codes[:, :, :8], cache.k_meta, cache.v_meta), lens)
    with pytest.raises(TypeError):
        ops.kv4_attn(q, cache, ints([3]))
    with pytest.raises(TypeError):
        ops.kv4_attn(q.half(), cache, lens)
    for bad in (dict(sm_scale=0.0), dict(sm_scale=math.inf), dict(sm_scale=1e300), dict(sm_scale=-1.0), dict(window=-1), dict(sinks=-1, window=4), dict(out=q)):
        with pytest.raises(L.Tb200Error):
            ops.kv4_attn(q, cache, lens, **bad)
    with pytest.raises(L.Tb200Error):       # three query heads on two key/value heads
        ops.kv4_attn(torch.zeros(2, 3, 1, 64, dtype=dt, device=DEV), cache, lens)
    with pytest.raises(L.Tb200Error):       # head_dim
        ops.attn_window(torch.zeros(1, 1, 1, 96, dtype=dt, device=DEV), torch.zeros(1, 1, 4, 96, dtype=dt, device=DEV),
                        torch.zeros(1, 1, 4, 96, dtype=dt, device=DEV), ints([1]))
    assert ops.device_status() == 0
