"""Attention over 16-bit and 4-bit caches against 64 bits, within a bound that follows the data (tests/cache_attn_bound.py):
long contexts, where the output is small beside the values, included.  Rows at the borders of tiles, windows and first
positions are sixteen times larger than the others; tests/test_cache_attn_bound.py shows what the bound notices."""
import pytest
import torch

from tests import cache_attn_bound as B
from tests.test_cache_attn_bound import SHAPES as CPU_SHAPES
from tests.test_gpu_cache_attn import SHAPES as GPU_SHAPES
from trinity_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16]
EPS16 = B.half_step(torch.float16)

# b, hq, hkv, d, s, cache length, lens, rows, window, sinks
SHAPES = GPU_SHAPES + CPU_SHAPES[-2:] + [
    (24, 32, 8, 128, 1, 3000, [3000 - 117 * i for i in range(24)], [1] * 24, 0, 0),
    (3, 32, 4, 128, 3, 20000, [20000, 7001, 13000], [3, 1, 2], 0, 0),
    (1, 16, 1, 64, 6, 33000, [32999], [6], 0, 0),
    (5, 24, 2, 128, 70, 5000, [5000, 70, 4097, 69, 1300], [70, 70, 1, 33, 64], 0, 0),
    (2, 40, 8, 64, 2, 17000, [17000, 16001], [2, 2], 9000, 63),
]


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def held4(k, v):
    """A 4-bit cache of the 16-bit rows k, v, and (k, v, weight of v) in 64 bits."""
    b, h, length, d = k.shape
    cache = ops.kv4_cache(b, h, length, d, k.dtype, DEV)
    wide = []
    for x, codes, meta in ((k, cache.k_codes, cache.k_meta), (v, cache.v_codes, cache.v_meta)):
        c, s, lo = B.quantise64(x)
        codes[:, :, :length], meta[:, :, :length] = B.pack4(c), torch.stack([s, lo], -1)
        wide.append(B.values64(codes[:, :, :length], meta[:, :, :length]))
    return cache, wide[0][0], wide[1][0], wide[1][1]


def run4(q, cache, k, v, w, lens, rows, window, sinks, scale):
    """kv4_attn and how far it is off, as a multiple of the bound."""
    b, hq, s, d = q.shape
    out = torch.full((b, s, hq, d), 7.0, dtype=q.dtype, device=DEV).transpose(1, 2)
    ops.kv4_attn(q, cache, ints(lens), window=window, sinks=sinks, sm_scale=scale, q_rows=ints(rows), out=out)
    assert ops.device_status() == 0
    prompt = s > 1 and s * hq // k.shape[1] > 64       # the form that rounds keys and values to 11 bits
    want, bound = B.attention_and_bound(q, k, v, lens, rows, window, sinks, scale, q.dtype, EPS16, weight=w * 2 ** 0.5 if prompt else w,
                                        eps_k=EPS16 if prompt else 0.0)
    return B.worst(out, want, bound)


def run16(q, k, v, lens, rows, window, sinks, scale):
    b, hq, s, d = q.shape
    out = torch.full((b, s, hq, d), 7.0, dtype=q.dtype, device=DEV).transpose(1, 2)
    ops.attn_window(q, k, v, ints(lens), window=window, sinks=sinks, sm_scale=scale, q_rows=ints(rows), out=out)
    assert ops.device_status() == 0
    want, bound = B.attention_and_bound(q, k.double(), v.double(), lens, rows, window, sinks, scale, q.dtype, B.half_step(q.dtype))
    return B.worst(out, want, bound)


def data(shape, dt, seed=5):
    b, hq, hkv, d, s, length, lens, rows, window, sinks = shape
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(b, s, hq, d, generator=g, device=DEV).to(dt).transpose(1, 2)
    k = (torch.randn(b, hkv, length, d, generator=g, device=DEV) + torch.randn(1, hkv, 1, d, generator=g, device=DEV)).to(dt)
    v = B.marked(torch.randn(b, hkv, length, d, generator=g, device=DEV), lens, rows, window, sinks).to(dt)
    return q, k, v


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_kv4_attn(shape, dt):
    q, k, v = data(shape, dt)
    assert run4(q, *held4(k, v), *shape[6:], shape[3] ** -0.5) <= 1


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attn_window(shape, dt):
    q, k, v = data(shape, dt)
    assert run16(q, k, v, *shape[6:], shape[3] ** -0.5) <= 1


@pytest.mark.parametrize("kv4", [True, False])
@pytest.mark.parametrize("s", [1, 3, 10, 40])
@pytest.mark.parametrize("e", [-120, -90, -64, 63, 64, 100, 107, 112, 120, 124])
def test_queries_and_keys_of_any_size(e, s, kv4):
    """bf16 queries 2^e times larger and keys as much smaller: the same scores.  One query row is of ordinary size, some keys
    are zeros."""
    shape = (2, 4, 1, 128, s, 512, [500, 77], [s, s], 0, 0)
    q, k, v = data(shape, torch.bfloat16)
    q, k = (q.float() * 2.0 ** e).to(q.dtype), (k.float() * 2.0 ** -e).to(k.dtype)
    q[0, 1, 0] = (q[0, 1, 0].float() * 2.0 ** -e).to(q.dtype) if e > 0 else q[0, 1, 0]
    k[:, :, 3::7] = 0
    off = run4(q, *held4(k, v), *shape[6:], 128 ** -0.5) if kv4 else run16(q, k, v, *shape[6:], 128 ** -0.5)
    assert off <= 1


@pytest.mark.parametrize("s", [1, 3, 10, 40])
@pytest.mark.parametrize("size", [1e30, 1e12, 1e-12, 1e-24, 1e-27, 1e-30, 1e-33])
def test_kv4_attn_values_of_any_size(size, s):
    """The products with V are fp16: V far from 1 altogether."""
    shape = (2, 4, 1, 128, s, 512, [500, 77], [s, s], 0, 0)
    q, k, v = data(shape, torch.bfloat16)
    assert run4(q, *held4(k, (v.float() * size).to(v.dtype)), *shape[6:], 128 ** -0.5) <= 1


@pytest.mark.parametrize("dt,s,first,second", [(torch.bfloat16, s, 1.0, x) for s in (1, 3, 10) for x in (1e6, 1e-4, 1e-6, 1e-9, 1e-24)]
                         + [(torch.float16, s, 100.0, x) for s in (1, 3, 10, 40) for x in (1.0, 1e-2, 1e-3)]
                         + [(torch.bfloat16, 40, 1.0, x) for x in (1e6, 1e-4, 1e-6)])
def test_kv4_attn_groups_of_unlike_size(dt, s, first, second):
    """64 channels of V many times smaller than the others keep their digits."""
    shape = (2, 4, 1, 128, s, 512, [500, 77], [s, s], 0, 0)
    q, k, v = data(shape, dt)
    v = torch.cat([v[..., :64].float() * first, v[..., 64:].float() * second], -1).to(dt)
    assert run4(q, *held4(k, v), *shape[6:], 128 ** -0.5) <= 1


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("s", [1, 3])
def test_kv4_attn_values_that_grow(s, dt):
    """Larger values the later a key comes: what has been summed is brought to the new scale, group by group."""
    shape = (1, 8, 2, 128, s, 12000, [11999], [s], 0, 0)
    q, k, v = data(shape, dt)
    grow = 2.0 ** torch.linspace(-10, 10 if dt == torch.bfloat16 else 6, 12000, device=DEV)
    f = v.float()
    f[..., :64] *= grow[:, None]
    f[..., 64:] *= grow.flip(0)[:, None]
    assert run4(q, *held4(k, f.to(dt)), *shape[6:], 128 ** -0.5) <= 1


@pytest.mark.parametrize("kv4", [True, False])
@pytest.mark.parametrize("s", [1, 3, 10, 40])
@pytest.mark.parametrize("scale", [1e-30, 1e-20, 1e20, 1e32, 1e37])
def test_scales_of_any_size(scale, s, kv4):
    """Queries as much smaller, or larger, as the scale is far from 1."""
    shape = (1, 4, 1, 128, s, 512, [500], [s], 0, 0)
    q, k, v = data(shape, torch.bfloat16)
    q = (q.float() * (128 ** -0.5 / scale)).to(q.dtype)
    off = run4(q, *held4(k, v), *shape[6:], scale) if kv4 else run16(q, k, v, *shape[6:], scale)
    assert off <= 1


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("s", [1, 3, 10, 40])
@pytest.mark.parametrize("e", [8, 12, 15, 20, 25])
def test_queries_with_one_large_channel(e, s, dt):
    """One channel of the queries 2^e times larger than the others, on keys that are zero there: the others keep their digits."""
    shape = (1, 4, 1, 128, s, 512, [500], [s], 0, 0)
    q, k, v = data(shape, dt)
    if dt == torch.float16:
        q = q * 2.0 ** -6      # (some of them below the type's smallest normal number)
    q[..., 5] = min(2.0 ** e, 60000.0) if dt == torch.float16 else 2.0 ** e
    k = k.abs()
    k[..., 5] = 0
    scale = 128 ** -0.5 * (64 if dt == torch.float16 else 1)
    cache, k64, v64, w = held4(k, v)
    assert (k64[..., 5] == 0).all()
    assert run4(q, cache, k64, v64, w, *shape[6:], scale) <= 1
