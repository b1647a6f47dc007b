"""Codes of the 4-bit cache against the definition in fp32: difference and quotient each rounded once, halves to even."""
import pytest
import torch

from trinity_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
CASES = [(torch.bfloat16, e) for e in (-133, -131, -129, -128, -127, -126, -125, -123, -121, -120, -119, -117, -100, -30, 0, 60, 118)] \
    + [(torch.float16, e) for e in (-24, -22, -20, -19, -18, -17, -14, -8, 0, 9)]


def quantise32(x):
    g = x.unflatten(-1, (-1, 64))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi.float() - lo.float()) / torch.full_like(hi, 15, dtype=torch.float32)).to(x.dtype)    # (a scalar divisor would become a factor 1/15)
    c = torch.where(s > 0, ((g.float() - lo.float()) / s.float()).round().clamp(0, 15), torch.zeros((), device=x.device))
    return c.flatten(-2), s.squeeze(-1), lo.squeeze(-1)


def appended(x):
    """Codes, s and lo that kv4_append leaves for the rows x (rows, 64)."""
    cache = ops.kv4_cache(1, 1, x.shape[0], 64, x.dtype, DEV)
    ops.kv4_append(cache, x[None, None], x[None, None], 0)
    for a, b in ((cache.k_codes, cache.v_codes), (cache.k_meta, cache.v_meta)):
        assert torch.equal(a, b)
    n = x.shape[0]
    codes = torch.stack([cache.k_codes & 15, cache.k_codes >> 4], -1).flatten(-2)[0, 0, :n].float()
    return codes, cache.k_meta[0, 0, :n, :, 0], cache.k_meta[0, 0, :n, :, 1]


@pytest.mark.parametrize("dt,e", CASES)
def test_codes_of_any_size(dt, e):
    """Whole numbers (many exact halves) and others times 2^e, some of them tiny beside the rest."""
    g = torch.Generator(device=DEV).manual_seed(e + 200)
    n = 1 << 15
    x = torch.randn(n, 64, generator=g, device=DEV, dtype=torch.float64) * 8
    x = torch.where(torch.rand(n, 64, generator=g, device=DEV) < 0.5, x.round(), x)
    x = torch.where(torch.rand(n, 64, generator=g, device=DEV) < 0.05, x * 2.0 ** -20, x) * 2.0 ** e
    x = x.clamp(-torch.finfo(dt).max / 4, torch.finfo(dt).max / 4).to(dt)
    for got, want in zip(appended(x), quantise32(x)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dt,tiny", [(torch.bfloat16, 1e-8), (torch.bfloat16, 1e-30), (torch.float16, 2.0 ** -24)])
def test_a_value_tiny_beside_the_minimum(dt, tiny):
    """lo = -15, s = 2: values around 0 lie in the middle between the codes 7 and 8, and get the even one on both sides."""
    x = torch.zeros(1, 64, dtype=torch.float64, device=DEV)
    x[0, 0], x[0, 1], x[0, 2], x[0, 3], x[0, 4:] = -15, 15, tiny, -tiny, 0
    codes, s, lo = appended(x.to(dt))
    assert s.item() == 2 and lo.item() == -15 and codes[0, 0] == 0 and codes[0, 1] == 15 and (codes[0, 2:] == 8).all()
