"""Cache rows that no query row of their sequence sees may hold anything: the same bits with zeros, NaN and infinities there, in
every kernel of attention over caches (tokens in clusters and on the line, drafts, prompts, ragged prompts; both caches)."""
import math

import pytest
import torch

from tests import cache_attn_bound as B
from tests.test_gpu_cache_attn_bound import DEV, TYPES, held4, ints
from trinity_b200 import ops

pytestmark = pytest.mark.gpu

# b, hq, hkv, s, cache length, lens, rows (None: no q_rows)
FORMS = {
    "clusters": (3, 8, 2, 1, 1200, [1100, 3, 700], [1, 1, 0]),
    "line": (40, 16, 8, 1, 700, [17 * i for i in range(40)], None),
    "long line": (3, 8, 4, 2, 9000, [9000, 1, 5003], [2, 2, 1]),
    "draft": (3, 16, 2, 7, 1200, [1200, 5, 800], [7, 7, 3]),
    "prompt": (1, 8, 2, 150, 1200, [1003], None),
    "prompts": (3, 4, 2, 150, 1200, [1003, 100, 0], None),
    "ragged prompts": (4, 4, 2, 150, 1200, [1003, 100, 40, 777], [150, 150, 0, 33]),
    "many ragged prompts": (130, 2, 1, 70, 400, [3 * i for i in range(130)], [i % 71 for i in range(130)]),
}


@pytest.mark.parametrize("window,sinks", [(0, 0), (130, 0), (130, 5), (100, 17), (64, 33), (300, 400)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("kv4", [True, False])
@pytest.mark.parametrize("form", FORMS)
def test_hidden_rows(form, kv4, dt, d, window, sinks):
    b, hq, hkv, s, length, lens, rows = FORMS[form]
    g = torch.Generator(device=DEV).manual_seed(6)
    q = torch.randn(b, hq, s, d, generator=g, device=DEV).to(dt)
    k, v = (torch.randn(b, hkv, length, d, generator=g, device=DEV).to(dt) for _ in range(2))
    live = torch.zeros(b, length, dtype=torch.bool, device=DEV)
    for i in range(b):
        n, r = B.clamped(lens[i], s if rows is None else rows[i], length, s)
        if r:
            live[i, :n] = B.visible(n, r, window, sinks, DEV).any(0)
    hidden = ~live[:, None].expand(b, hkv, length)
    cache = held4(k, v)[0] if kv4 else None
    kw = dict(window=window, sinks=sinks, sm_scale=0.1, q_rows=None if rows is None else ints(rows))
    outs = []
    for fill in (0.0, math.nan, math.inf, -math.inf):
        if kv4:
            for codes, meta in ((cache.k_codes, cache.k_meta), (cache.v_codes, cache.v_meta)):
                codes[hidden], meta[hidden] = 0x5a, fill
            outs.append(ops.kv4_attn(q, cache, ints(lens), **kw))
        else:
            k[hidden], v[hidden] = fill, fill
            outs.append(ops.attn_window(q, k, v, ints(lens), **kw))
    assert ops.device_status() == 0 and torch.isfinite(outs[0]).all()
    for x in outs[1:]:
        assert torch.equal(x, outs[0])
