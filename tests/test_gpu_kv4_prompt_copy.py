"""Prompts on a 4-bit cache compute on a 16-bit copy of what is visible: its size, the pieces in which a large call is done, and
what lies in the scratch memory between the rows."""
import ctypes as C

import pytest
import torch

from tests import cache_attn_bound as B
from tests.test_gpu_cache_attn_bound import DEV, EPS16, TYPES, ints
from trinity_b200 import _lib as L
from trinity_b200 import ops

pytestmark = pytest.mark.gpu
MIB = 1 << 20


def workspace_bytes(b, hq, hkv, d, s, length, window, sinks, dtype=L.BF16):
    a = L.CacheAttnArgs(dtype=dtype, batch=b, rows=s, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, cache_len=length, window=window, sinks=sinks, sm_scale=0.1,
                        q=0x1000, o=0x2000, q_stride=(C.c_int64 * 3)(hq * s * d, s * d, d), o_stride=(C.c_int64 * 3)(hq * s * d, s * d, d), kv_lens=0x3000,
                        k_codes=0x4000, v_codes=0x5000, k_meta=0x6000, v_meta=0x7000)
    return L.load().tb200_kv4_attn_workspace_bytes(C.byref(a))


@pytest.mark.parametrize("b,hq,hkv,d,s,length,window,sinks,most", [
    (24, 32, 8, 128, 500, 16384, 0, 0, 256 * MIB),       # the copy of the whole cache would be 1536 MiB
    (24, 32, 8, 128, 20, 16384, 0, 0, 256 * MIB),
    (16, 32, 8, 128, 20, 131072, 0, 0, 1024 * MIB),      # 8192 MiB
    (2, 4, 2, 128, 100, 1 << 22, 0, 0, 2048 * MIB),      # one (sequence, kv head) at a time
    (16, 32, 8, 128, 20, 131072, 1000, 4, 16 * 8 * (1000 + 20 + 16) * 128 * 4),
    (1, 8, 1, 64, 500, 1 << 28, 200, 17, (200 + 500 + 32) * 64 * 4),
])
def test_scratch_is_bounded_and_follows_what_is_visible(b, hq, hkv, d, s, length, window, sinks, most):
    """Besides the copy: q in fp16, its powers of two, partial results of shared keys (at most 16 shares of fewer rows than SMs
    have)."""
    rest = b * hq * s * (2 * d + 4) + 16 * 74 * 256 * (d + 2) * 4 + b * hkv * 16 + 4096
    assert workspace_bytes(b, hq, hkv, d, s, length, window, sinks) <= most + rest


def long_cache(b, h, length, d, dt, at, seed=3):
    """A cache of `length` positions that holds rows at the given positions only, and those rows in 64 bits (with the weight of
    v); the rest is NaN."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    cache = ops.Kv4Cache(*[torch.full((b, h, length, d // 2), 255, dtype=torch.uint8, device=DEV) for _ in range(2)],
                         *[torch.full((b, h, length, d // 64, 2), float("nan"), dtype=dt, device=DEV) for _ in range(2)])
    wide = []
    for codes, meta in ((cache.k_codes, cache.k_meta), (cache.v_codes, cache.v_meta)):
        x = (torch.randn(b, h, len(at), d, generator=g, device=DEV) + torch.randn(1, h, 1, d, generator=g, device=DEV)).to(dt)
        c, s, lo = B.quantise64(x)
        codes[:, :, at], meta[:, :, at] = B.pack4(c), torch.stack([s, lo], -1)
        wide.append(B.values64(codes[:, :, at], meta[:, :, at]))
    return cache, wide[0][0], wide[1][0], wide[1][1]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("b,hq,hkv,s,length,lens,rows", [
    (3, 8, 4, 40, 400_000, [700, 64, 333], [40, 33, 40]),        # pieces of two sequences and of one
    (2, 12, 3, 40, 3_000_000, [600, 41], [40, 17]),              # of one (sequence, kv head)
    (1, 10, 5, 40, 1_500_000, [500], [40]),                      # of two kv heads and of one
])
def test_pieces(b, hq, hkv, s, length, lens, rows, dt):
    d, scale = 64, 64 ** -0.5
    n = max(lens)
    cache, k, v, w = long_cache(b, hkv, length, d, dt, torch.arange(n, device=DEV))
    one = length * d * 4                                         # bytes of the copy of one (sequence, kv head)
    assert workspace_bytes(b, hq, hkv, d, s, length, 0, 0) < b * hkv * one
    g = torch.Generator(device=DEV).manual_seed(1)
    q = torch.randn(b, s, hq, d, generator=g, device=DEV).to(dt).transpose(1, 2)
    out = torch.full((b, s, hq, d), 7.0, dtype=dt, device=DEV).transpose(1, 2)
    lens_, rows_ = ints(lens), ints(rows)
    call = lambda: ops.kv4_attn(q, cache, lens_, sm_scale=scale, q_rows=rows_, out=out)
    call()
    want, bound = B.attention_and_bound(q, k, v, lens, rows, 0, 0, scale, dt, EPS16, weight=w * 2 ** 0.5, eps_k=EPS16)
    assert B.worst(out, want, bound) <= 1
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    out.fill_(7)
    graph.replay()
    assert torch.equal(out, first) and ops.device_status() == 0


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(100, 0), (100, 5), (257, 16), (130, 33), (1, 1)])
def test_a_window_far_into_a_long_cache(window, sinks, d, dt):
    """Only the first positions and the window hold anything; the copy is of their size.  A second sequence ends before its
    window begins, a third has no rows."""
    length, s, hq, hkv, scale = 2_000_000, 150, 4, 2, d ** -0.5
    n, r = length - 5, [150, 150, 0]
    tail = n - r[0] - window + 1
    at = torch.cat([torch.arange(200, device=DEV), torch.arange(tail, n, device=DEV)])
    cache, k, v, w = long_cache(3, hkv, length, d, dt, at)
    assert workspace_bytes(3, hq, hkv, d, s, length, window, sinks) < 3 * hkv * (window + s + 64) * d * 4 + 3 * hq * s * (2 * d + 4) + 16 * 74 * 256 * (d + 2) * 4
    g = torch.Generator(device=DEV).manual_seed(1)
    q = torch.randn(3, hq, s, d, generator=g, device=DEV).to(dt)
    out = torch.full_like(q, 7.0)
    ops.kv4_attn(q, cache, ints([n, 160, n]), window=window, sinks=sinks, sm_scale=scale, q_rows=ints(r), out=out)
    # the long sequence without what lies between the first positions and the window: each row sees what it saw
    few = torch.cat([torch.arange(sinks, device=DEV), torch.arange(200, at.numel(), device=DEV)])
    for i, (keys, m) in enumerate(((few, few.numel()), (torch.arange(200, device=DEV), 160))):
        args = [t[i:i + 1, :, keys] for t in (k, v, w)]
        want, bound = B.attention_and_bound(q[i:i + 1], args[0], args[1], [m], [s], window, sinks, scale, dt, EPS16, weight=args[2] * 2 ** 0.5, eps_k=EPS16)
        assert B.worst(out[i:i + 1], want, bound) <= 1
    assert torch.equal(out[2], torch.full_like(out[2], 7.0)) and ops.device_status() == 0


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,s,lens,rows,window,sinks", [
    (1, 130, [700], None, 0, 0), (1, 130, [900], None, 200, 5), (2, 130, [900, 333], [130, 77], 150, 33), (3, 70, [64, 900, 5], [70, 70, 3], 0, 0),
    (2, 300, [900, 900], None, 100, 17), (1, 40, [1000], None, 500, 12)])
def test_what_the_scratch_held_before_does_not_matter(b, s, lens, rows, window, sinks, d, dt):
    """The same bits with NaN in all of the scratch memory, and with zeros."""
    g = torch.Generator(device=DEV).manual_seed(2)
    cache = ops.kv4_cache(b, 2, 1000, d, dt, DEV)
    x = torch.randn(b, 2, 1000, d, generator=g, device=DEV).to(dt)
    ops.kv4_append(cache, x, x.flip(2).contiguous(), 0)
    q = torch.randn(b, 8, s, d, generator=g, device=DEV).to(dt)
    kw = dict(window=window, sinks=sinks, sm_scale=0.1, q_rows=None if rows is None else ints(rows))
    outs = []
    ops.kv4_attn(q, cache, ints(lens), **kw)                     # sizes the workspace
    held = [t for key, t in ops.Workspace._bufs.items() if key[1] == "tb200_kv4_attn"]
    assert held
    for fill in (0, 255):
        for t in held:
            t.fill_(fill)
        outs.append(ops.kv4_attn(q, cache, ints(lens), **kw))
    assert torch.isfinite(outs[0]).all() and torch.equal(outs[0], outs[1])
