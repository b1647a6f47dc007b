"""Tensor-level wrappers over the C ABI: torch tensors in, raw device pointers across the boundary.

PyTorch is plumbing here (device memory, streams); every operator below runs in libtrinity_b200.so.
All wrappers launch on ``torch.cuda.current_stream()`` and allocate nothing once their workspace has
been cached (attention over caches: but for a 16-bit copy of a large 4-bit cache, and in a capture, where
scratch comes out of the graph's pool), so they can be captured in a CUDA graph after one warm-up call.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Dict, NamedTuple, Optional, Union

import torch

from . import _lib as L

_DT = {torch.float16: L.F16, torch.bfloat16: L.BF16, torch.float32: L.F32}


def _dt(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("trinity_b200 operators take CUDA tensors (there is no CPU path)")
    if not t.is_contiguous():
        raise ValueError("trinity_b200 operators take contiguous tensors")
    return t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


_current_raw_stream = torch._C._cuda_getCurrentRawStream


def _raw_stream(index: int) -> int:
    """The current stream of device `index`, without a Stream object (which costs about 3 us)."""
    return _current_raw_stream(index)


class Workspace:
    """Scratch buffers the operators hand to the C ABI, one per (device, tag, stream).

    * A buffer only grows, and only outside CUDA-graph capture (the first call sizes it).
    * A buffer that is outgrown is RETIRED, not freed: a CUDA graph captured earlier holds its device address, and
      the caching allocator must not hand that memory to another tensor while the graph can still be replayed.
      ``Workspace.release()`` drops the retired buffers once no such graph is left.
    * Buffers are keyed by the stream the call runs on, so eager calls on two streams never share partial sums; the
      memory is allocated on that stream, so the allocator's stream bookkeeping is right without ``record_stream``.
    * A capture on a stream that has no buffer yet adopts the one a warm-up call sized on another stream (capture
      cannot allocate).  The two streams then share it: do not run that warm-up stream while the graph replays.
    """

    _bufs: Dict[tuple, torch.Tensor] = {}
    _retired: list = []

    @classmethod
    def get(cls, device: torch.device, nbytes: int, tag: str = "default") -> Optional[torch.Tensor]:
        if nbytes == 0:
            return None
        index = device.index if device.index is not None else torch.cuda.current_device()
        key = (index, tag, _raw_stream(index))
        buf = cls._bufs.get(key)
        if buf is None or buf.numel() < nbytes:
            if torch.cuda.is_current_stream_capturing():
                for (i, t, _), other in cls._bufs.items():
                    if i == index and t == tag and other.numel() >= nbytes:
                        if buf is not None:
                            cls._retired.append(buf)
                        cls._bufs[key] = other
                        return other
                raise RuntimeError("workspace must be sized by one call outside CUDA-graph capture first")
            if buf is not None:
                cls._retired.append(buf)
            buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
            cls._bufs[key] = buf
        return buf

    @classmethod
    def release(cls) -> None:
        """Free the buffers that were outgrown.  Call only when no CUDA graph captured before the growth is replayed again."""
        cls._retired.clear()


class FoldedWeights:
    """Projection weights with an RMSNorm weight folded into their rows (``tb200_fold_norm_weight``), kept per set of
    source tensors.  ``(x * r * g) @ W = r * (x @ (diag(g) W))``: with the folded copy the weighted norm in front of a
    projection is a row statistic and a per-row scale in the projection's epilogue, no normalised copy of ``x``.

    A folded copy is made at the first call that sees a (weights, norm weight) combination -- outside CUDA-graph
    capture, like any one-time set-up; under capture an unseen combination runs the unfolded path -- and reused while
    the source tensors are alive and unmodified (their torch version counters are part of the key).  It costs the
    projection's weight bytes once more in HBM; ``FoldedWeights.enabled = False`` turns folding off."""

    enabled = True
    _cache: Dict[tuple, tuple] = {}

    @classmethod
    def get(cls, g: torch.Tensor, *weights: torch.Tensor):
        if not cls.enabled:
            return None
        key = (g.data_ptr(), g._version) + tuple((w.data_ptr(), w._version, tuple(w.shape)) for w in weights)
        hit = cls._cache.get(key)
        if hit is not None:
            return hit[0]
        if torch.cuda.is_current_stream_capturing():
            return None
        lib = L.load()
        folded = []
        for w in weights:
            out = torch.empty_like(w)
            L.check(lib.tb200_fold_norm_weight(_ptr(w), _ptr(g), _ptr(out), w.shape[0], w.shape[1], _dt(w), _stream()), "tb200_fold_norm_weight")
            folded.append(out)
        if len(cls._cache) >= 64:          # a bound, not a policy: drop the oldest entry
            cls._cache.pop(next(iter(cls._cache)))
        cls._cache[key] = (tuple(folded), (g,) + weights)   # the sources are kept alive so that their addresses stay theirs
        return tuple(folded)

    @classmethod
    def clear(cls) -> None:
        cls._cache.clear()


def rmsnorm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 0.0,
            out: Optional[torch.Tensor] = None, inv_rms: Optional[torch.Tensor] = None) -> torch.Tensor:
    lib = L.load()
    cols = x.shape[-1]
    rows = x.numel() // cols
    if out is None:
        out = torch.empty_like(x)
    L.check(lib.tb200_rmsnorm(_ptr(x), _ptr(weight), _ptr(out), _ptr(inv_rms), rows, cols, eps, _dt(x), _stream()), "tb200_rmsnorm")
    return out


def row_inv_rms(x: torch.Tensor, eps: float = 0.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Only the per-row statistic ``rsqrt(mean(x^2) + eps)`` (fp32), for the norm-as-epilogue path."""
    lib = L.load()
    cols = x.shape[-1]
    rows = x.numel() // cols
    if out is None:
        out = torch.empty(rows, dtype=torch.float32, device=x.device)
    L.check(lib.tb200_rmsnorm(_ptr(x), None, None, _ptr(out), rows, cols, eps, _dt(x), _stream()), "tb200_rmsnorm")
    return out


def gemm(a: torch.Tensor, b: torch.Tensor, *, b2: Optional[torch.Tensor] = None, row_scale: Optional[torch.Tensor] = None,
         residual: Optional[torch.Tensor] = None, act: int = 0, split_k: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    lib = L.load()
    m, k = a.shape
    n = b.shape[1]
    if out is None:
        out = torch.empty(m, n, dtype=a.dtype, device=a.device)
    args = L.GemmArgs(dtype=_dt(a), act=act, m=m, n=n, k=k, a=_ptr(a), b=_ptr(b), b2=_ptr(b2), c=_ptr(out),
                      row_scale=_ptr(row_scale), residual=_ptr(residual), split_k=split_k)
    need = lib.tb200_gemm_workspace_bytes(C.byref(args))
    ws = Workspace.get(a.device, need, "gemm")
    args.workspace, args.workspace_bytes = _ptr(ws), need
    L.check(lib.tb200_gemm(C.byref(args), _stream()), "tb200_gemm")
    return out


def _attn_args(x, wq, wk, wv, k_cache, v_cache, o2, *, past: int, head_dim: int, flags: int = 0,
               sm_scale: float = 1.0, norm_weight=None, norm_eps: float = 0.0, q_norm_weight=None,
               k_norm_weight=None, qk_eps: float = 0.0, noise=None, tau: float = 1.5, c_out=None,
               c_out1=None, c_out2=None, topk: int = 0, topk_idx=None):
    """The argument block of tb200_attn_forward with its workspace attached.  Returns (args, tensors to keep alive)."""
    lib = L.load()
    if x.dim() == 2:
        batch, (seq, hidden) = 1, x.shape
    else:
        batch, seq, hidden = x.shape
    n_q = wq.shape[1] // head_dim
    n_kv = wk.shape[1] // head_dim
    cache_len = k_cache.shape[-2]
    if (flags & L.ATTN_PRENORM) and norm_weight is not None and not (flags & L.ATTN_NORM_FOLDED):
        folded = FoldedWeights.get(norm_weight, wq, wk, wv)
        if folded is not None:
            wq, wk, wv = folded
            flags |= L.ATTN_NORM_FOLDED
    aux = c_out if c_out is not None else c_out1
    args = L.AttnArgs(
        dtype=_dt(x), flags=flags, batch=batch, seq=seq, hidden=hidden, n_q_heads=n_q, n_kv_heads=n_kv,
        head_dim=head_dim, past=past, cache_len=cache_len, sm_scale=sm_scale, norm_eps=norm_eps, qk_eps=qk_eps, tau=tau,
        x=_ptr(x), wq=_ptr(wq), wk=_ptr(wk), wv=_ptr(wv), k_cache=_ptr(k_cache), v_cache=_ptr(v_cache), o2=_ptr(o2),
        norm_weight=_ptr(norm_weight), q_norm_weight=_ptr(q_norm_weight), k_norm_weight=_ptr(k_norm_weight),
        noise=_ptr(noise), c_out=_ptr(c_out), c_out1=_ptr(c_out1), c_out2=_ptr(c_out2),
        aux_dtype=_dt(aux) if aux is not None else L.F32, topk=topk, topk_idx=_ptr(topk_idx))
    need = lib.tb200_attn_workspace_bytes(C.byref(args))
    if need == 0:
        raise L.Tb200Error(-1, "tb200_attn_workspace_bytes")
    ws = Workspace.get(x.device, need, "attn")
    args.workspace, args.workspace_bytes = _ptr(ws), need
    return args, (wq, wk, wv, ws)


def attn_forward(*tensors, timed: bool = False, **kw):
    """The fused attention block: ``attn_forward(x, wq, wk, wv, k_cache, v_cache, o2, past=, head_dim=, flags=, ...)``;
    mutates ``o2``, the cache rows ``[past, past+S)`` and the c_out* tensors.  With ``timed`` the call waits for the
    stream and returns the four stage durations in ms."""
    lib = L.load()
    args, _keep = _attn_args(*tensors, **kw)
    if timed:
        ms = (C.c_float * 4)()
        L.check(lib.tb200_attn_forward_timed(C.byref(args), _stream(), ms), "tb200_attn_forward_timed")
        return list(ms)
    L.check(lib.tb200_attn_forward(C.byref(args), _stream()), "tb200_attn_forward")


def _ffn_args(x, w_gate, w_up, w_down, ff2, *, act: int = L.FFN_SWIGLU, flags: int = 0, o2=None, wo=None,
              norm_weight=None, norm_eps: float = 0.0, tail_divisor: int = 0, attn_o2=None, ff1=None,
              o_ff_norm=None):
    """The argument block of tb200_ffn_forward with its workspace attached.  Returns (args, tensors to keep alive)."""
    lib = L.load()
    hidden = x.shape[-1]
    tokens = x.numel() // hidden
    inner = w_gate.shape[1]
    if (flags & L.FFN_NORM) and norm_weight is not None and not (flags & (L.FFN_NORM_FOLDED | L.FFN_FALCON_TAIL)):
        folded = FoldedWeights.get(norm_weight, *([w_gate] if w_up is None else [w_gate, w_up]))
        if folded is not None:
            w_gate, w_up = folded[0], (folded[1] if w_up is not None else None)
            flags |= L.FFN_NORM_FOLDED
    args = L.FfnArgs(dtype=_dt(x), act=act, flags=flags, tokens=tokens, hidden=hidden, inner=inner, norm_eps=norm_eps,
                     tail_divisor=tail_divisor, x=_ptr(x), o2=_ptr(o2), wo=_ptr(wo), norm_weight=_ptr(norm_weight),
                     w_gate=_ptr(w_gate), w_up=_ptr(w_up), w_down=_ptr(w_down), ff2=_ptr(ff2), attn_o2=_ptr(attn_o2),
                     ff1=_ptr(ff1), o_ff_norm=_ptr(o_ff_norm))
    need = lib.tb200_ffn_workspace_bytes(C.byref(args))
    ws = Workspace.get(x.device, need, "ffn")
    args.workspace, args.workspace_bytes = _ptr(ws), need
    return args, (w_gate, w_up, ws)


def ffn_forward(*tensors, **kw) -> None:
    """The fused FFN block: ``ffn_forward(x, w_gate, w_up, w_down, ff2, act=, flags=, o2=, wo=, ...)``; mutates ``ff2``
    (and ``attn_o2`` / ``ff1`` / ``o_ff_norm`` when given)."""
    args, _keep = _ffn_args(*tensors, **kw)
    L.check(L.load().tb200_ffn_forward(C.byref(args), _stream()), "tb200_ffn_forward")


def layer_forward(attn: dict, ffn: dict) -> None:
    """The attention block and the FFN block that consumes its ``o2`` as ONE call (tb200_layer_forward): one launch chain,
    in which the FFN's first projection starts its weight stream while the attention kernel drains.  ``attn`` and ``ffn``
    hold the arguments of ``attn_forward`` / ``ffn_forward`` (positional tensors under the key ``"tensors"``); the FFN's
    ``o2`` must be the attention block's."""
    a_args, _ka = _attn_args(*attn["tensors"], **{k: v for k, v in attn.items() if k != "tensors"})
    f_args, _kf = _ffn_args(*ffn["tensors"], **{k: v for k, v in ffn.items() if k != "tensors"})
    L.check(L.load().tb200_layer_forward(C.byref(a_args), C.byref(f_args), _stream()), "tb200_layer_forward")


def topk(scores: torch.Tensor, k: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    lib = L.load()
    n = scores.shape[-1]
    rows = scores.numel() // n
    if out is None:
        out = torch.empty(*scores.shape[:-1], k, dtype=torch.int32, device=scores.device)
    L.check(lib.tb200_topk(_ptr(scores), _ptr(out), rows, n, k, _stream()), "tb200_topk")
    return out


def kv_compact(k_src: torch.Tensor, v_src: torch.Tensor, idx: torch.Tensor, kv_len: int, keep_recent: int = 0,
               k_dst: Optional[torch.Tensor] = None, v_dst: Optional[torch.Tensor] = None, kept_pos: Optional[torch.Tensor] = None,
               new_len: Optional[torch.Tensor] = None):
    """Pack the cache positions ``idx`` names (and the last ``keep_recent``) to the front of ``k_dst`` / ``v_dst``.

    ``k_src, v_src``: ``(..., L, D)`` caches, leading axes = batch and kv heads; ``idx``: int32 ``(..., n_idx)`` over the
    same leading axes.  Returns ``(k_dst, v_dst, kept_pos, new_len)``; destination caches are allocated
    ``(..., max_keep, D)`` when not given; ``k_dst=k_src, v_dst=v_src`` packs in place."""
    lib = L.load()
    if idx.dtype != torch.int32:
        raise TypeError("idx must be int32")
    if k_src.shape != v_src.shape or k_src.dtype != v_src.dtype:
        raise ValueError("k_src and v_src must agree in shape and dtype")
    lead = k_src.shape[:-2]
    if tuple(idx.shape[:-1]) != tuple(lead):
        raise ValueError(f"idx leading axes {tuple(idx.shape[:-1])} do not match the caches' {tuple(lead)}")
    rows = 1
    for d in lead:
        rows *= int(d)
    args = L.KvCompactArgs(dtype=_dt(k_src), rows=rows, head_dim=int(k_src.shape[-1]), kv_len=int(kv_len),
                           src_cache_len=int(k_src.shape[-2]), n_idx=int(idx.shape[-1]), keep_recent=int(keep_recent))
    max_keep = int(lib.tb200_kv_compact_max_keep(C.byref(args)))
    dev = k_src.device
    if k_dst is None:
        k_dst = torch.empty(*lead, max_keep, k_src.shape[-1], dtype=k_src.dtype, device=dev)
    if v_dst is None:
        v_dst = torch.empty(*lead, max_keep, k_src.shape[-1], dtype=k_src.dtype, device=dev)
    if k_dst.shape != v_dst.shape or k_dst.dtype != k_src.dtype or v_dst.dtype != k_src.dtype:
        raise ValueError("k_dst and v_dst must agree in shape and share the source dtype")
    if tuple(k_dst.shape[:-2]) != tuple(lead) or k_dst.shape[-1] != k_src.shape[-1]:
        raise ValueError("destination caches must have the source's leading axes and head dimension")
    if kept_pos is None:
        kept_pos = torch.empty(*lead, max_keep, dtype=torch.int32, device=dev)
    if new_len is None:
        new_len = torch.empty(*lead, dtype=torch.int32, device=dev)
    if kept_pos.dtype != torch.int32 or new_len.dtype != torch.int32 or kept_pos.numel() != rows * max_keep or new_len.numel() != rows:
        raise ValueError("kept_pos must be int32 (..., max_keep) and new_len int32 (...)")
    args.dst_cache_len = int(k_dst.shape[-2])
    args.idx, args.k_src, args.v_src = _ptr(idx), _ptr(k_src), _ptr(v_src)
    args.k_dst, args.v_dst, args.kept_pos, args.new_len = _ptr(k_dst), _ptr(v_dst), _ptr(kept_pos), _ptr(new_len)
    L.check(lib.tb200_kv_compact(C.byref(args), _stream()), "tb200_kv_compact")
    return k_dst, v_dst, kept_pos, new_len


class Kv4Cache(NamedTuple):
    """A KV cache in 4 bits: groups of 64 values of a row as codes ``c`` of 4 bits and a pair ``(s, lo)`` of the cache's
    16-bit type, standing for ``lo + c * s`` (include/trinity_b200.h has the definition).

    ``k_codes, v_codes``: uint8 ``(B, Hkv, L, D / 2)``, element ``2 i`` in the low and ``2 i + 1`` in the high four bits
    of byte ``i``; ``k_meta, v_meta``: ``(B, Hkv, L, D / 64, 2)``.  ``L`` is a multiple of 4."""
    k_codes: torch.Tensor
    v_codes: torch.Tensor
    k_meta: torch.Tensor
    v_meta: torch.Tensor


def kv4_cache(batch: int, kv_heads: int, cache_len: int, head_dim: int, dtype: torch.dtype = torch.bfloat16, device="cuda") -> Kv4Cache:
    """An empty 4-bit cache of at least ``cache_len`` positions (rounded up to a multiple of 4); ``head_dim`` 64 or 128,
    ``dtype`` bfloat16 or float16."""
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, not {head_dim}")
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"a 4-bit cache stands for bfloat16 or float16 rows, not {dtype}")
    if cache_len < 0:
        raise ValueError(f"cache_len must not be negative, not {cache_len}")
    length = (cache_len + 3) // 4 * 4
    codes = [torch.zeros(batch, kv_heads, length, head_dim // 2, dtype=torch.uint8, device=device) for _ in range(2)]
    meta = [torch.zeros(batch, kv_heads, length, head_dim // 64, 2, dtype=dtype, device=device) for _ in range(2)]
    return Kv4Cache(*codes, *meta)


# The argument blocks of L.Kv4RowsArgs and L.CacheAttnArgs, packed in one call and handed over as bytes: a ctypes structure
# filled field by field costs more than the launch of a small kernel.
_KV4_ROWS = struct.Struct("@8i2P2P3q3q4P")
_CACHE_ATTN = struct.Struct("@9if2P3q3q2P2P3q3q4PPN")
assert _KV4_ROWS.size == C.sizeof(L.Kv4RowsArgs) and _CACHE_ATTN.size == C.sizeof(L.CacheAttnArgs)
_ENTRIES: dict = {}


def _entry(name: str, restype=C.c_int, argtypes=(C.c_char_p, C.c_void_p)):
    """A function of the library that takes its argument block as bytes."""
    f = _ENTRIES.get(name)
    if f is None:
        f = L.load()[name]     # (an object of its own: the one behind the attribute takes the structure)
        f.restype, f.argtypes = restype, argtypes
        _ENTRIES[name] = f
    return f


def _refuse_rows(t: torch.Tensor, name: str, shape, dtype: torch.dtype, index: int):
    if not t.is_cuda:
        raise ValueError("trinity_b200 operators take CUDA tensors (there is no CPU path)")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, the call's first tensor on cuda:{index}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, not {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    raise ValueError(f"the last axis of {name} must be contiguous")


def _rows4(t: torch.Tensor, name: str, shape, dtype: torch.dtype, index: int):
    """Strides of a ``(B, heads, rows, D)`` tensor whose last axis is contiguous, in elements."""
    if t.dtype is dtype and t.shape == shape and t.get_device() == index:
        strides = t.stride()
        if strides[3] == 1:
            return strides
    _refuse_rows(t, name, shape, dtype, index)


def _ints(t: Optional[torch.Tensor], name: str, batch: int, index: int) -> int:
    if t is None:
        return 0
    if t.__class__ is torch.Tensor and t.dtype is torch.int32 and t.shape == (batch,) and t.get_device() == index and t.is_contiguous():
        return t.data_ptr()
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.shape != (batch,):
        raise TypeError(f"{name} must be an int32 tensor of shape ({batch},)")
    if t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor on cuda:{index}")
    return t.data_ptr()


def _kv4_parts(cache: Kv4Cache, index: int):
    """(batch, kv heads, cache length, head_dim, type) of a 4-bit cache."""
    kc, vc, km, vm = cache
    shape, dt = kc.shape, km.dtype
    if len(shape) != 4:
        raise ValueError(f"k_codes must have shape (B, Hkv, L, D / 2), not {tuple(shape)}")
    b, h, length, half = shape
    meta = (b, h, length, half // 32, 2)
    if not (kc.dtype is torch.uint8 and vc.dtype is torch.uint8 and vm.dtype is dt and vc.shape == shape and km.shape == meta and vm.shape == meta
            and half % 32 == 0):
        raise ValueError(f"codes must be uint8 (B, Hkv, L, D / 2), meta 16-bit (B, Hkv, L, D / 64, 2), alike for k and v; not "
                         + ", ".join(f"{t.dtype} {tuple(t.shape)}" for t in cache))
    if not (kc.get_device() == vc.get_device() == km.get_device() == vm.get_device() == index
            and kc.is_contiguous() and vc.is_contiguous() and km.is_contiguous() and vm.is_contiguous()):
        raise ValueError(f"the parts of a 4-bit cache must be contiguous tensors on cuda:{index}")
    return b, h, length, 2 * half, dt


def _device_index(t: torch.Tensor) -> int:
    index = t.get_device()
    if index < 0:
        raise ValueError("trinity_b200 operators take CUDA tensors (there is no CPU path)")
    return index


_current_device = torch._C._cuda_getDevice


def _kv4_rows(name: str, cache: Kv4Cache, k, v, start, rows, index: int, count: Optional[int] = None) -> None:
    b, h, length, d, dt = _kv4_parts(cache, index)
    if count is None:
        count = k.shape[2] if k.dim() == 4 else -1
    shape = (b, h, count, d)
    ks, vs = _rows4(k, "k", shape, dt, index), _rows4(v, "v", shape, dt, index)
    one = isinstance(start, int)
    if start is None:
        raise TypeError("start must be an int or an int32 tensor")
    kc, vc, km, vm = cache
    try:
        packed = _KV4_ROWS.pack(
            _dt(k), b, h, count, d, length, start if one else 0, 0, 0 if one else _ints(start, "start", b, index), _ints(rows, "rows", b, index),
            k.data_ptr(), v.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], kc.data_ptr(), vc.data_ptr(), km.data_ptr(), vm.data_ptr())
    except struct.error as e:
        raise ValueError(f"an argument is no whole number or out of range: {e}") from None
    if index == _current_device():
        status = _entry(name)(packed, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = _entry(name)(packed, _raw_stream(index))
    if status:
        L.check(status, name)


def kv4_append(cache: Kv4Cache, k: torch.Tensor, v: torch.Tensor, start: Union[int, torch.Tensor], rows: Optional[torch.Tensor] = None) -> None:
    """Quantise new rows into a 4-bit cache: row ``i`` of ``k, v (B, Hkv, S, D)`` becomes position ``start[b] + i``.

    ``k`` and ``v`` may have any strides that are multiples of 8 and at least ``D`` (last axis contiguous): what a projection leaves,
    ``(x @ wk).view(B, S, Hkv, D).transpose(1, 2)``, needs no copy.  ``start``: an int for all sequences or int32 ``(B,)``;
    ``rows`` int32 ``(B,)``: how many of the ``S`` rows of each sequence are meant (default all).  Other rows, and rows
    whose position lies outside the cache, are not written."""
    _kv4_rows("tb200_kv4_append", cache, k, v, start, rows, _device_index(k))


def kv4_read(cache: Kv4Cache, start: Union[int, torch.Tensor], count: int, rows: Optional[torch.Tensor] = None,
             k_out: Optional[torch.Tensor] = None, v_out: Optional[torch.Tensor] = None):
    """Rows ``[start[b], start[b] + count)`` of a 4-bit cache as 16-bit rows ``(B, Hkv, count, D)``: ``lo + c * s`` rounded
    once (at most the type's largest number).  ``rows`` int32 ``(B,)`` limits how many are read of each sequence; the
    others, and positions outside the cache, are left as they are in ``k_out, v_out`` (zero when these are not given).
    Returns ``(k_out, v_out)``."""
    index = _device_index(cache.k_codes)
    if k_out is None or v_out is None:
        b, h, _, half = cache.k_codes.shape
        make = lambda: torch.zeros(b, h, count, 2 * half, dtype=cache.k_meta.dtype, device=cache.k_codes.device)
        k_out = make() if k_out is None else k_out
        v_out = make() if v_out is None else v_out
    _kv4_rows("tb200_kv4_read", cache, k_out, v_out, start, rows, index, count)
    return k_out, v_out


_KEPT_SCRATCH = 64 << 20   # decode calls need a few MB
_NEEDS_WORKSPACE = -4      # TB200_ERR_WORKSPACE
_WORKSPACE = struct.Struct("@PN")   # the end of _CACHE_ATTN


def _cache_attn(name: str, q, out, kv_lens, q_rows, window, sinks, sm_scale, dims, caches, index: int):
    if index != _current_device():
        with torch.cuda.device(index):
            return _cache_attn(name, q, out, kv_lens, q_rows, window, sinks, sm_scale, dims, caches, index)
    b, h, length, d, dt = dims
    if kv_lens is None:
        raise TypeError("kv_lens must be an int32 tensor")
    try:
        _, hq, s, _ = q.shape
    except ValueError:
        raise ValueError(f"q must have shape (B, Hq, S, D), not {tuple(q.shape)}") from None
    if out is None:
        out = torch.empty(b, s, hq, d, dtype=dt, device=q.device).transpose(1, 2)
        if q_rows is not None:
            out.zero_()
    shape = (b, hq, s, d)
    qs, os_ = _rows4(q, "q", shape, dt, index), _rows4(out, "out", shape, dt, index)
    try:
        packed = _CACHE_ATTN.pack(
            _dt(q), b, s, hq, h, d, length, window, sinks, sm_scale, q.data_ptr(), out.data_ptr(), qs[0], qs[1], qs[2], os_[0], os_[1], os_[2],
            _ints(kv_lens, "kv_lens", b, index), _ints(q_rows, "q_rows", b, index), *caches, 0, 0)
    except struct.error as e:
        raise ValueError(f"an argument is no whole number or out of range: {e}") from None
    status = _entry(name)(packed, _raw_stream(index))
    if status == _NEEDS_WORKSPACE:   # nothing has been launched; calls on short caches need none
        need = _entry(name + "_workspace_bytes", C.c_size_t, (C.c_char_p,))(packed)
        # a graph gets scratch of its own, out of its memory pool: graphs captured on one stream may run side by side.  A 16-bit
        # copy of a large cache is not kept between calls.
        own = need > _KEPT_SCRATCH or torch._C._cuda_isCurrentStreamCapturing()
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if own else Workspace.get(q.device, need, name)
        status = _entry(name)(packed[:-_WORKSPACE.size] + _WORKSPACE.pack(ws.data_ptr(), need), _raw_stream(index))
    if status:
        L.check(status, name)
    return out


def attn_window(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, kv_lens: torch.Tensor, *, window: int = 0, sinks: int = 0,
                sm_scale: float = 1.0, q_rows: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``softmax(sm_scale * q K^T) V`` over 16-bit caches that already hold the new rows, with per-sequence lengths.

    ``q (B, Hq, S, D)``, ``k_cache, v_cache (B, Hkv, L, D)``: any strides that are multiples of 8 and at least ``D`` (last axis
    contiguous).
    ``kv_lens`` int32 ``(B,)``: positions in the cache, the new ones included; ``q_rows`` int32 ``(B,)``: how many of the
    ``S`` query rows belong to the sequence (default all); they are the last positions.  A query sees the positions up to
    its own, with ``window > 0`` only the last ``window`` of these and the first ``sinks`` ones.  A row that sees nothing
    gives zeros.  Rows from ``q_rows`` on are left as they are in ``out`` (zero when it is not given).  ``out`` overlaps
    none of the inputs.  Returns ``out``, ``(B, Hq, S, D)``; by default laid out so that
    ``out.transpose(1, 2).reshape(B, S, Hq * D)`` is a view.  Forward only."""
    index = _device_index(q)
    shape = k_cache.shape
    if len(shape) != 4:
        raise ValueError(f"k_cache must have shape (B, Hkv, L, D), not {tuple(shape)}")
    ks, vs = _rows4(k_cache, "k_cache", shape, q.dtype, index), _rows4(v_cache, "v_cache", shape, q.dtype, index)
    caches = (k_cache.data_ptr(), v_cache.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], 0, 0, 0, 0)
    return _cache_attn("tb200_attn_window", q, out, kv_lens, q_rows, window, sinks, sm_scale, (*shape, q.dtype), caches, index)


def kv4_attn(q: torch.Tensor, cache: Kv4Cache, kv_lens: torch.Tensor, *, window: int = 0, sinks: int = 0, sm_scale: float = 1.0,
             q_rows: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``attn_window`` over a 4-bit cache: the same arguments and the same result, with ``cache`` a :class:`Kv4Cache`."""
    index = _device_index(q)
    dims = _kv4_parts(cache, index)
    kc, vc, km, vm = cache
    caches = (0, 0, 0, 0, 0, 0, 0, 0, kc.data_ptr(), vc.data_ptr(), km.data_ptr(), vm.data_ptr())
    return _cache_attn("tb200_kv4_attn", q, out, kv_lens, q_rows, window, sinks, sm_scale, dims, caches, index)


def device_status() -> int:
    """Synchronise and return the device error word (0 = healthy); raises on a recorded timeout."""
    code = C.c_int(0)
    status = L.load().tb200_device_status(C.byref(code))
    if status != 0:
        raise L.Tb200Error(status, f"tb200_device_status (device code {code.value})")
    return code.value
