"""Workloads of the 4-bit KV cache and of windowed attention: inputs, plain form, 64-bit form and work of each case.

Four operators, all on caches of the shape (batch, kv heads, positions, head_dim):

  kv4_write    new key and value rows are quantised into a 4-bit cache as they are written, then read back
  kv4_read     rows of a 4-bit cache are read back as 16-bit rows
  kv4_attn     softmax(sm_scale * q K^T) V over a 4-bit cache, for single tokens and for prompts
  attn_window  the same over a 16-bit cache, each query seeing a sliding window and the first few positions

The 4-bit form of 64 consecutive values x of a row (a group): lo = min x, s = (max x - min x) / 15, both kept in the
cache's 16-bit type, c = the whole number nearest to (x - lo) / s in [0, 15] (0 where s is 0; halves go to the even one).
A group stands for lo + c * s.  Codes lie two to a byte, the even element in the low four bits; meta holds (s, lo).

A query in row i of r new rows of a sequence of n positions stands at position n - r + i and sees the positions up to its
own; with a window w it sees of those the last w and the first `sinks` ones.
"""
import math
import random

import torch

own = False

GROUP = 64
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_CHUNK = 512   # queries of a prompt handled at a time by the plain form


def listed():
    return [
        # one decoding step's new rows of eight sequences: all launch latency
        {"name": "write_token", "op": "kv4_write", "batch": 8, "kv_heads": 8, "q_heads": 32, "head_dim": 128, "dtype": "bf16",
         "cache_len": 2048, "rows": 1, "ragged": True, "window": 0, "sinks": 0},
        # the prompts of a ragged batch on their way into the cache
        {"name": "write_prompts", "op": "kv4_write", "batch": 8, "kv_heads": 8, "q_heads": 32, "head_dim": 128, "dtype": "bf16",
         "cache_len": 4096, "rows": 4093, "ragged": True, "window": 0, "sinks": 0},
        # a short stretch of one multi-query cache
        {"name": "read_short", "op": "kv4_read", "batch": 1, "kv_heads": 1, "q_heads": 71, "head_dim": 64, "dtype": "f16",
         "cache_len": 1040, "rows": 1037, "ragged": False, "window": 0, "sinks": 0},
        # whole caches handed back to 16-bit code
        {"name": "read_long", "op": "kv4_read", "batch": 8, "kv_heads": 8, "q_heads": 32, "head_dim": 128, "dtype": "f16",
         "cache_len": 8192, "rows": 8192, "ragged": True, "window": 0, "sinks": 0},
        # a single user's next token on a short context: latency
        {"name": "token_short", "op": "kv4_attn", "batch": 1, "kv_heads": 8, "q_heads": 32, "head_dim": 128, "dtype": "bf16",
         "cache_len": 1040, "rows": 1, "ragged": False, "window": 0, "sinks": 0},
        # a served batch with contexts of very different lengths
        {"name": "token_batch", "op": "kv4_attn", "batch": 24, "kv_heads": 8, "q_heads": 32, "head_dim": 128, "dtype": "bf16",
         "cache_len": 16384, "rows": 1, "ragged": True, "window": 0, "sinks": 0},
        # 71 query heads on one key/value head, long contexts
        {"name": "token_mqa_long", "op": "kv4_attn", "batch": 4, "kv_heads": 1, "q_heads": 71, "head_dim": 64, "dtype": "f16",
         "cache_len": 65536, "rows": 1, "ragged": False, "window": 0, "sinks": 0},
        # a few proposed tokens checked at once, window and first tokens
        {"name": "draft_window", "op": "kv4_attn", "batch": 16, "kv_heads": 8, "q_heads": 32, "head_dim": 128, "dtype": "f16",
         "cache_len": 8192, "rows": 5, "ragged": True, "window": 2048, "sinks": 4},
        # the next piece of a long prompt on a 4-bit cache
        {"name": "prompt_piece", "op": "kv4_attn", "batch": 1, "kv_heads": 8, "q_heads": 32, "head_dim": 128, "dtype": "bf16",
         "cache_len": 4096, "rows": 500, "ragged": False, "window": 0, "sinks": 0},
        # streaming decoding of a batch
        {"name": "window_token", "op": "attn_window", "batch": 32, "kv_heads": 8, "q_heads": 32, "head_dim": 128, "dtype": "bf16",
         "cache_len": 4096, "rows": 1, "ragged": True, "window": 1024, "sinks": 4},
        # a whole prompt under a window
        {"name": "window_prompt", "op": "attn_window", "batch": 1, "kv_heads": 8, "q_heads": 32, "head_dim": 128, "dtype": "bf16",
         "cache_len": 4000, "rows": 4000, "ragged": False, "window": 1000, "sinks": 4},
        # a ragged batch of prompts on one key/value head each
        {"name": "window_prompts_mha", "op": "attn_window", "batch": 3, "kv_heads": 16, "q_heads": 16, "head_dim": 64, "dtype": "f16",
         "cache_len": 1800, "rows": 1111, "ragged": True, "window": 300, "sinks": 17},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    most = {"kv4_write": 3.5e8, "kv4_read": 3.5e8, "kv4_attn": 3.0e8, "attn_window": 2.5e8}
    while True:
        op = rng.choice(["kv4_write", "kv4_read", "kv4_attn", "kv4_attn", "attn_window", "attn_window"])
        head_dim = rng.choice([64, 128, 128])
        kv_heads = rng.choice([1, 2, 4, 8, 16])
        group = rng.choice([1, 2, 4, 4, 7, 8, 16]) if kv_heads > 1 else rng.choice([1, 8, 32, 71])
        batch = _spread(rng, 1, 32)
        length = _spread(rng, 16, 65536 if op == "kv4_attn" else 8192)
        if op == "kv4_write":
            rows = rng.choice([1, 1, _spread(rng, 2, length)])
        elif op == "kv4_read":
            rows = _spread(rng, 1, length)
        else:
            rows = min(length, rng.choice([1, 1, _spread(rng, 2, 16), _spread(rng, 17, 2048)]))
        window = sinks = 0
        if op == "attn_window" or rng.random() < 0.3:
            window, sinks = _spread(rng, 16, 4096), rng.choice([0, 1, 4, 16, 33])
        case = {"op": op, "batch": batch, "kv_heads": kv_heads, "q_heads": kv_heads * group, "head_dim": head_dim,
                "dtype": rng.choice(["bf16", "f16"]), "cache_len": (length + 3) // 4 * 4, "rows": rows, "ragged": rng.random() < 0.5,
                "window": window, "sinks": sinks}
        if op in ("kv4_write", "kv4_read"):
            case["window"] = case["sinks"] = 0
        cached = batch * kv_heads * case["cache_len"] * head_dim   # values of one of the two caches
        w = work(case)
        if cached <= 2.0e8 and w["bytes"] <= most[op] and w["flops"] <= 5e10:
            return case


def _lens(case):
    """Positions of each sequence (the new ones included) and new rows of each."""
    rng = random.Random(case["batch"] * 1000003 + case["cache_len"] * 31 + case["rows"])
    n, r = [], []
    for b in range(case["batch"]):
        if case["ragged"]:
            rows = case["rows"] if case["rows"] < 17 or b == 0 else rng.randint(1, case["rows"])
            n.append(rng.randint(max(rows, case["cache_len"] // 8), case["cache_len"]))
            r.append(rows)
        else:
            n.append(case["cache_len"] - (3 if case["cache_len"] - case["rows"] > 2 else 0))
            r.append(case["rows"])
    return n, r


def _pairs(n, r, window, sinks):
    """(query, key) pairs that are visible, and the keys that some query sees, of one sequence."""
    if not window:
        return r * n - r * (r - 1) // 2, n
    pairs = 0
    for i in range(r):
        at = n - r + i
        low = max(0, at - window + 1)
        pairs += at + 1 - low + min(sinks, low)
    low = max(0, n - r - window + 1)
    return pairs, n - low + min(sinks, low)


def work(case):
    n, r = _lens(case)
    heads, d = case["kv_heads"], case["head_dim"]
    row4 = d // 2 + d // GROUP * 4           # bytes of one 4-bit row: codes and (s, lo) of each group
    row16 = 2 * d
    if case["op"] == "kv4_write":            # 16-bit rows in, 4-bit rows out and in again, 16-bit rows out; K and V
        rows = sum(r) * heads
        return {"bytes": 2 * rows * (2 * row16 + 2 * row4), "flops": 2 * rows * d * 8}
    if case["op"] == "kv4_read":
        rows = sum(r) * heads
        return {"bytes": 2 * rows * (row16 + row4), "flops": 2 * rows * d * 2}
    pairs = keys = 0
    for a, b in zip(n, r):
        p, k = _pairs(a, b, case["window"], case["sinks"])
        pairs, keys = pairs + p, keys + k
    row = row4 if case["op"] == "kv4_attn" else row16
    return {"bytes": 2 * keys * heads * row + 2 * sum(r) * case["q_heads"] * row16, "flops": 4 * pairs * case["q_heads"] * d}


# ---------------------------------------------------------------------------------------------- the 4-bit form
def _quantise(x):
    """x (..., d) 16-bit -> codes (..., d) uint8, meta (..., d / 64, 2) of x's type."""
    g = x.unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi.float() - lo.float()) / 15).to(x.dtype)
    # the quotient in 64 bits: values next to a border between two codes
    t = (g.double() - lo.double()) / s.double()
    c = torch.where(s > 0, t.round().clamp(0, 15), torch.zeros_like(t)).to(torch.uint8)
    return c.flatten(-2), torch.cat([s, lo], -1)


def _pack(c):
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _unpack(p):
    return torch.stack([p & 15, p >> 4], -1).flatten(-2)


def _values(codes, meta):
    """What a packed cache stands for, in 32 bits."""
    c = _unpack(codes).unflatten(-1, (-1, GROUP)).float()
    return (meta[..., 1:].float() + c * meta[..., :1].float()).flatten(-2)


def _new_rows(case, gen):
    """Keys lie around an offset of their channel, values around zero."""
    d, heads = case["head_dim"], case["kv_heads"]
    shape = (case["batch"], case["rows"], heads, d)
    dt = _TYPES[case["dtype"]]
    k = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * 0.7 + torch.randn((heads, d), generator=gen, device="cuda")
    v = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return k.to(dt).transpose(1, 2), v.to(dt).transpose(1, 2)   # (batch, heads, rows, d) as a projection leaves them


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[case["dtype"]]
    b, heads, length, d = case["batch"], case["kv_heads"], case["cache_len"], case["head_dim"]
    n, r = _lens(case)
    st = {"case": case, "n": n, "r": r}
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    st["lens"], st["rows"], st["start"] = ints(n), ints(r), ints([x - y for x, y in zip(n, r)])
    if case["op"] != "attn_window":
        codes = [torch.empty(b, heads, length, d // 2, dtype=torch.uint8, device="cuda") for _ in range(2)]
        meta = [torch.empty(b, heads, length, d // GROUP, 2, dtype=dt, device="cuda") for _ in range(2)]
        for i in range(2):
            off = torch.randn((heads, 1, d), generator=gen, device="cuda") * (1 - i)
            for j in range(b):
                x = torch.randn((heads, length, d), generator=gen, device="cuda") * (0.7 + 0.3 * i) + off
                c, m = _quantise(x.to(dt))
                codes[i][j], meta[i][j] = _pack(c), m
        st["k_codes"], st["v_codes"], st["k_meta"], st["v_meta"] = codes[0], codes[1], meta[0], meta[1]
    else:
        off = torch.randn((heads, 1, d), generator=gen, device="cuda")
        st["k_cache"] = (torch.randn((b, heads, length, d), generator=gen, device="cuda") * 0.7 + off).to(dt)
        st["v_cache"] = torch.randn((b, heads, length, d), generator=gen, device="cuda").to(dt)
    if case["op"] == "kv4_write":
        st["k"], st["v"] = _new_rows(case, gen)
    if case["op"] in ("kv4_write", "kv4_read"):
        st["k_out"] = torch.zeros(b, heads, case["rows"], d, dtype=dt, device="cuda")
        st["v_out"] = torch.zeros_like(st["k_out"])
    else:
        q = torch.randn((b, case["rows"], case["q_heads"], d), generator=gen, device="cuda")
        st["q"] = q.to(dt).transpose(1, 2)
        st["out"] = torch.zeros(b, case["rows"], case["q_heads"], d, dtype=dt, device="cuda").transpose(1, 2)
        st["scale"] = d ** -0.5
    return st


# ---------------------------------------------------------------------------------------------- the plain forms
def _plain_write(st):
    for j, (n, r) in enumerate(zip(st["n"], st["r"])):
        for x, codes, meta, out in ((st["k"], st["k_codes"], st["k_meta"], st["k_out"]), (st["v"], st["v_codes"], st["v_meta"], st["v_out"])):
            c, m = _quantise(x[j, :, :r])
            codes[j, :, n - r:n], meta[j, :, n - r:n] = _pack(c), m
            out[j, :, :r] = _values(codes[j, :, n - r:n], meta[j, :, n - r:n]).to(out.dtype)
    return st["k_out"], st["v_out"]


def _plain_read(st):
    for j, (n, r) in enumerate(zip(st["n"], st["r"])):
        for codes, meta, out in ((st["k_codes"], st["k_meta"], st["k_out"]), (st["v_codes"], st["v_meta"], st["v_out"])):
            out[j, :, :r] = _values(codes[j, :, n - r:n], meta[j, :, n - r:n]).to(out.dtype)
    return st["k_out"], st["v_out"]


def _plain_attention(st):
    case = st["case"]
    window, sinks, heads = case["window"], case["sinks"], case["kv_heads"]
    for j, (n, r) in enumerate(zip(st["n"], st["r"])):
        first = max(0, n - r - window + 1) if window else 0
        first = 0 if first <= sinks else first
        parts = [slice(0, n)] if first == 0 else [slice(0, sinks), slice(first, n)]
        at = torch.cat([torch.arange(p.start, p.stop, device="cuda") for p in parts])
        if case["op"] == "kv4_attn":
            k = torch.cat([_values(st["k_codes"][j, :, p], st["k_meta"][j, :, p]) for p in parts], 1)
            v = torch.cat([_values(st["v_codes"][j, :, p], st["v_meta"][j, :, p]) for p in parts], 1)
        else:
            k = torch.cat([st["k_cache"][j, :, p] for p in parts], 1).float()
            v = torch.cat([st["v_cache"][j, :, p] for p in parts], 1).float()
        k, v = k.unsqueeze(1), v.unsqueeze(1)
        q = st["q"][j].unflatten(0, (heads, -1)).float()              # (kv heads, group, rows, d)
        out = st["out"][j].unflatten(0, (heads, -1))
        for i in range(0, r, _CHUNK):
            e = min(r, i + _CHUNK)
            pos = torch.arange(n - r + i, n - r + e, device="cuda").unsqueeze(1)
            # the keys between the first query's window and the last query's position, and the first few
            low = max(0, n - r + i - window + 1) if window else 0
            low = low - first + sinks if first else low               # its place in `at`
            high = len(at) - (r - e)
            few = min(sinks, low)
            take = lambda t: t[:, :, low:high] if not few else torch.cat([t[:, :, :few], t[:, :, low:high]], 2)
            key = at[low:high] if not few else torch.cat([at[:few], at[low:high]])
            seen = key <= pos
            if window:
                seen &= (key > pos - window) | (key < sinks)
            s = (q[:, :, i:e] @ take(k).transpose(-1, -2)) * st["scale"]
            s = torch.where(seen, s, torch.full((), -math.inf, device="cuda"))
            s = torch.exp(s - s.amax(-1, keepdim=True))
            out[:, :, i:e] = ((s @ take(v)) / s.sum(-1, keepdim=True)).to(out.dtype)
    return st["out"]


# ---------------------------------------------------------------------------------------------- the framework's calls
def _own(st):
    from trinity_b200 import ops
    case = st["case"]
    if case["op"] == "attn_window":
        return ops.attn_window(st["q"], st["k_cache"], st["v_cache"], st["lens"], window=case["window"], sinks=case["sinks"],
                               sm_scale=st["scale"], q_rows=st["rows"], out=st["out"])
    cache = ops.Kv4Cache(st["k_codes"], st["v_codes"], st["k_meta"], st["v_meta"])
    if case["op"] == "kv4_write":
        ops.kv4_append(cache, st["k"], st["v"], st["start"], rows=st["rows"])
    if case["op"] in ("kv4_write", "kv4_read"):
        return ops.kv4_read(cache, st["start"], case["rows"], rows=st["rows"], k_out=st["k_out"], v_out=st["v_out"])
    return ops.kv4_attn(st["q"], cache, st["lens"], window=case["window"], sinks=case["sinks"], sm_scale=st["scale"],
                        q_rows=st["rows"], out=st["out"])


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "kv4_write":
        return _plain_write(state)
    if op == "kv4_read":
        return _plain_read(state)
    return _plain_attention(state)


# ---------------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_groups(x):
    """What the rows x stand for once they are held in 4 bits."""
    g = x.reshape(x.shape[:-1] + (x.shape[-1] // GROUP, GROUP)).double()
    lo = g.min(-1, keepdim=True).values
    s = ((g.max(-1, keepdim=True).values - lo) / 15).to(x.dtype).double()
    steps = torch.round((g - lo) / torch.where(s == 0, torch.ones_like(s), s))
    return (lo + torch.clamp(steps, 0, 15) * s).reshape(x.shape)


def _exact_rows(codes, meta, first, last):
    p = codes[:, first:last].to(torch.int64)
    c = torch.empty(p.shape[:-1] + (2 * p.shape[-1],), dtype=torch.float64, device=p.device)
    c[..., 0::2] = (p % 16).double()
    c[..., 1::2] = (p // 16).double()
    m = meta[:, first:last].double().repeat_interleave(GROUP, dim=2)
    return m[..., 1] + c * m[..., 0]


def exact(case, seed):
    st = prepare(case, seed)
    op, heads, d = case["op"], case["kv_heads"], case["head_dim"]
    if op in ("kv4_write", "kv4_read"):
        outs = []
        for i, name in enumerate(("k", "v")):
            out = torch.zeros(case["batch"], heads, case["rows"], d, dtype=torch.float64, device="cuda")
            for j in range(case["batch"]):
                n, r = st["n"][j], st["r"][j]
                if op == "kv4_write":
                    out[j, :, :r] = _exact_groups(st[name][j, :, :r])
                else:
                    out[j, :, :r] = _exact_rows(st[name + "_codes"][j], st[name + "_meta"][j], n - r, n)
            outs.append(out)
        return tuple(outs)
    group = case["q_heads"] // heads
    res = torch.zeros(case["batch"], case["q_heads"], case["rows"], d, dtype=torch.float64, device="cuda")
    for j in range(case["batch"]):
        n, r = st["n"][j], st["r"][j]
        key = torch.arange(n, device="cuda")[None, :]
        at = torch.arange(n - r, n, device="cuda")[:, None]
        hidden = key > at
        if case["window"]:
            hidden |= (at - key >= case["window"]) & (key >= case["sinks"])
        for h in range(heads):
            if op == "kv4_attn":
                k = _exact_rows(st["k_codes"][j, h:h + 1], st["k_meta"][j, h:h + 1], 0, n)[0]
                v = _exact_rows(st["v_codes"][j, h:h + 1], st["v_meta"][j, h:h + 1], 0, n)[0]
            else:
                k, v = st["k_cache"][j, h, :n].double(), st["v_cache"][j, h, :n].double()
            for a in range(group):
                z = torch.mm(st["q"][j, h * group + a, :r].double(), k.t()) * st["scale"]
                z.masked_fill_(hidden, -math.inf)
                res[j, h * group + a, :r] = torch.softmax(z, dim=1) @ v
    return res
