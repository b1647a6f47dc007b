"""The bound that the attention tests over caches use notices what a wrong kernel would do (no GPU): for every shape, results
with a part left out, a window of another length or a key too few lie outside of it, and one with rounded probabilities inside."""
import pytest
import torch

from tests import cache_attn_bound as B

# b, hq, hkv, d, s, cache length, lens, rows, window, sinks
SHAPES = [
    (3, 8, 2, 128, 1, 300, [300, 77, 129], [1, 1, 1], 0, 0),
    (2, 14, 2, 128, 1, 4096, [4001, 333], [1, 1], 128, 4),
    (2, 32, 8, 128, 5, 1000, [999, 400], [5, 2], 200, 16),
    (2, 8, 2, 64, 257, 1024, [1021, 600], [257, 100], 100, 4),
    (2, 6, 2, 128, 260, 1200, [1111, 300], [260, 260], 128, 300),
    (1, 2, 1, 128, 40, 20000, [19999], [40], 5000, 128),
    (2, 8, 2, 128, 1, 30000, [30000, 777], [1, 1], 0, 0),
    (2, 12, 2, 64, 2, 40000, [40000, 20011], [2, 2], 0, 0),
    (1, 20, 2, 128, 1, 24000, [23999], [1], 12000, 100),
    (1, 71, 1, 64, 1, 60000, [60000], [1], 0, 0),
    (1, 16, 4, 128, 130, 2100, [2100], [130], 0, 0),
]


def data(shape, dt, kv4):
    b, hq, hkv, d, s, length, lens, rows, window, sinks = shape
    g = torch.Generator().manual_seed(5)
    q = torch.randn(b, hq, s, d, generator=g).to(dt)
    k = (torch.randn(b, hkv, length, d, generator=g) + torch.randn(1, hkv, 1, d, generator=g)).to(dt)
    v = B.marked(torch.randn(b, hkv, length, d, generator=g), lens, rows, window, sinks).to(dt)
    if not kv4:
        return q, k.double(), v.double(), None
    held = []
    for x in (k, v):
        c, sc, lo = B.quantise64(x)
        held.append(B.values64(B.pack4(c), torch.stack([sc, lo], -1)))
    return q, held[0][0], held[1][0], held[1][1]


@pytest.mark.parametrize("kv4", [False, True])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_wrong_results_lie_outside_the_bound(shape, dt, kv4):
    b, hq, hkv, d, s, length, lens, rows, window, sinks = shape
    scale = d ** -0.5
    q, k, v, w = data(shape, dt, kv4)
    prompt = kv4 and s > 1 and s * hq // hkv > 64      # keys and values are rounded too: the widest bound of a 4-bit cache
    eps16 = B.half_step(torch.float16)
    want, bound = B.attention_and_bound(q, k, v, lens, rows, window, sinks, scale, dt, eps16 if kv4 else B.half_step(dt),
                                        weight=w * 2 ** 0.5 if prompt else w, eps_k=eps16 if prompt else 0.0)

    def off(seen_by):
        return B.worst(B.attention64(q, k, v, lens, rows, window, sinks, scale, seen_by), want, bound)

    def without(first, last):
        """No key of [first, last) of the sequence that is n - 1 long at most."""
        def seen_by(n, r, *a):
            seen = B.visible(n, r, *a)
            if n == max(lens):
                seen[:, first:last] = False
            return seen
        return seen_by

    assert off(B.visible) < 1e-6
    zeros = want.clone()
    for i in range(b):
        zeros[i, :, :rows[i]] = 0
    assert B.worst(zeros, want, bound) > 2
    n = max(lens)
    tile = 64 if kv4 else 16
    assert off(without(n - tile, n - s)) > 1.2 if n - tile < n - s else True     # the last tile but for the rows' own keys
    assert off(without(n - window // 2 if window else n // 2 // tile * tile, (n - window // 2 if window else n // 2 // tile * tile) + tile)) > 1.2
    own = lambda n, r, win, few, dev: B.visible(n, r, win, few, dev) & (torch.arange(n, device=dev)[None] != torch.arange(n - r, n, device=dev)[:, None])
    assert off(own) > 1.2
    if window:
        assert off(lambda n, r, win, few, dev: B.visible(n, r, win + 1, few, dev)) > 1.2
        assert off(lambda n, r, win, few, dev: B.visible(n, r, win - 1, few, dev)) > 1.2
        assert off(lambda n, r, win, few, dev: B.visible(n, r, win, 0, dev)) > 1.2
        assert off(lambda n, r, win, few, dev: B.visible(n, r, win, few - 1, dev)) > 1.2
        assert off(lambda n, r, win, few, dev: B.visible(n, r, win, few + 1, dev)) > 1.2


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES[:7], ids=str)
def test_rounded_probabilities_lie_inside(shape, dt):
    """The arithmetic of the 16-bit kernels: fp32 probabilities relative to the maximum, rounded, summed before that."""
    b, hq, hkv, d, s, length, lens, rows, window, sinks = shape
    scale = d ** -0.5
    q, k, v, _ = data(shape, dt, False)
    want, bound = B.attention_and_bound(q, k, v, lens, rows, window, sinks, scale, dt, B.half_step(dt))
    got = torch.full_like(want, 7.0).to(dt)
    for i in range(b):
        n, r = lens[i], rows[i]
        seen = B.visible(n, r, window, sinks, "cpu")
        z = (q[i, :, :r].float().unflatten(0, (hkv, hq // hkv)) @ k[i, :, None, :n].float().transpose(-1, -2)) * scale
        z = z.masked_fill(~seen, -float("inf"))
        p = torch.exp(z - z.amax(-1, keepdim=True))
        got[i, :, :r] = ((p.to(dt).float() @ v[i, :, None, :n].float()) / p.sum(-1, keepdim=True)).flatten(0, 1).to(dt)
    assert B.worst(got, want, bound) < 1
