"""Host-side argument checks of the 4-bit cache and of attention over caches: fake addresses, nothing is launched."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from trinity_b200 import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, UNSUPPORTED = -1, -2


@pytest.fixture(scope="module")
def lib():
    from trinity_b200 import build
    build.build()
    return L.load()


def rows_args(**kw):
    a = dict(dtype=L.BF16, batch=2, n_kv_heads=4, rows=16, head_dim=128, cache_len=64, k=0x1000, v=0x2000,
             k_stride=(8192, 2048, 128), v_stride=(8192, 128, 512), k_codes=0x3000, v_codes=0x4000, k_meta=0x5000, v_meta=0x6000)
    a.update(kw)
    for n in ("k_stride", "v_stride"):
        a[n] = (C.c_int64 * 3)(*a[n])
    return L.Kv4RowsArgs(**a)


def attn_args(**kw):
    a = dict(dtype=L.F16, batch=2, rows=3, n_q_heads=8, n_kv_heads=2, head_dim=64, cache_len=64, window=16, sinks=4, sm_scale=0.125,
             q=0x1000, o=0x2000, q_stride=(1536, 192, 64), o_stride=(1536, 64, 512), kv_lens=0x3004, k_cache=0x4000, v_cache=0x5000,
             k_stride=(8192, 4096, 64), v_stride=(8192, 64, 128), k_codes=0x6000, v_codes=0x7000, k_meta=0x8000, v_meta=0x9000)
    a.update(kw)
    for n in ("q_stride", "o_stride", "k_stride", "v_stride"):
        a[n] = (C.c_int64 * 3)(*a[n])
    return L.CacheAttnArgs(**a)


@pytest.mark.parametrize("change,status", [
    ({}, 0), (dict(dtype=L.F32), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED), (dict(batch=-1), INVALID), (dict(rows=-1), INVALID),
    (dict(n_kv_heads=0), INVALID), (dict(cache_len=62), INVALID), (dict(cache_len=-4), INVALID), (dict(reserved=1), INVALID), (dict(k=None), INVALID),
    (dict(v_meta=None), INVALID), (dict(k=0x1008), INVALID), (dict(k_codes=0x3008), INVALID), (dict(start=0x3002), INVALID),
    (dict(k_stride=(8192, 2048, 132)), INVALID), (dict(k_stride=(8192, 0, 128)), INVALID), (dict(k_stride=(8192, 2048, -128)), INVALID),
    (dict(rows=1, k_stride=(8192, 2048, 3)), 0), (dict(batch=0), 0), (dict(rows=0), 0), (dict(start=0x3004, n_rows=0x3008), 0)])
def test_rows_check(lib, change, status):
    assert lib.tb200_kv4_rows_check(C.byref(rows_args(**change))) == status
    if status:
        assert lib.tb200_kv4_append(C.byref(rows_args(**change)), None) == status
        assert lib.tb200_kv4_read(C.byref(rows_args(**change)), None) == status


def test_read_refuses_rows_that_overlap(lib):
    for stride in ((2048, 2048, 128), (8192, 128, 128), (8192, 1024, 128)):
        assert lib.tb200_kv4_read(C.byref(rows_args(k_stride=stride)), None) == INVALID
        assert lib.tb200_kv4_rows_check(C.byref(rows_args(k_stride=stride))) == 0      # as a source they may


def test_two_outputs_in_one_place_are_refused(lib):
    assert lib.tb200_kv4_read(C.byref(rows_args(v=0x1000)), None) == INVALID
    for same in (dict(v_codes=0x3000), dict(v_meta=0x5000)):
        assert lib.tb200_kv4_append(C.byref(rows_args(**same)), None) == INVALID
        assert lib.tb200_kv4_rows_check(C.byref(rows_args(**same))) == 0      # one cache for both may be read


@pytest.mark.parametrize("change", [dict(rows=(1 << 30) + 1), dict(cache_len=(1 << 30) + 4), dict(batch=(1 << 30) + 1), dict(n_kv_heads=(1 << 30) + 1)])
def test_rows_extents_are_bounded(lib, change):
    assert lib.tb200_kv4_rows_check(C.byref(rows_args(**change))) == INVALID


COMMON = [
    ({}, 0), (dict(dtype=L.F32), UNSUPPORTED), (dict(head_dim=256), UNSUPPORTED), (dict(n_q_heads=9), INVALID), (dict(n_q_heads=0), INVALID),
    (dict(cache_len=0), INVALID), (dict(window=-1), INVALID), (dict(sinks=-1), INVALID), (dict(sm_scale=0.0), INVALID), (dict(sm_scale=float("nan")), INVALID),
    (dict(sm_scale=float("inf")), INVALID), (dict(q=None), INVALID), (dict(o=0x1000), INVALID), (dict(o=0x2004), INVALID), (dict(kv_lens=None), INVALID),
    (dict(kv_lens=0x3002), INVALID), (dict(q_rows=0x3002), INVALID), (dict(o_stride=(1536, 64, 64)), INVALID), (dict(q_stride=(1536, 192, 60)), INVALID),
    (dict(o_stride=(512, 64, 512)), INVALID), (dict(batch=0), 0), (dict(rows=0), 0), (dict(q_rows=0x3008), 0)]


@pytest.mark.parametrize("change,status", COMMON + [
    (dict(k_cache=None), INVALID), (dict(v_cache=0x5008), INVALID), (dict(k_stride=(8192, 4096, 68)), INVALID), (dict(v_stride=(8192, 64, 32)), INVALID),
    (dict(cache_len=63), 0), (dict(k_codes=None), 0)])
def test_attn_window_check(lib, change, status):
    assert lib.tb200_attn_window_check(C.byref(attn_args(**change))) == status
    if status:
        assert lib.tb200_attn_window(C.byref(attn_args(**change)), None) == status


@pytest.mark.parametrize("change,status", COMMON + [
    (dict(k_codes=None), INVALID), (dict(v_meta=0x9008), INVALID), (dict(cache_len=62), INVALID), (dict(k_cache=None), 0)])
def test_kv4_attn_check(lib, change, status):
    assert lib.tb200_kv4_attn_check(C.byref(attn_args(**change))) == status
    if status:
        assert lib.tb200_kv4_attn(C.byref(attn_args(**change)), None) == status


def test_null_arguments(lib):
    for name in ("tb200_kv4_append", "tb200_kv4_read", "tb200_attn_window", "tb200_kv4_attn"):
        assert getattr(lib, name)(None, None) == INVALID
    for name in ("tb200_kv4_rows_check", "tb200_attn_window_check", "tb200_kv4_attn_check"):
        assert getattr(lib, name)(None) == INVALID
    assert lib.tb200_kv4_attn_workspace_bytes(None) == 0 and lib.tb200_attn_window_workspace_bytes(None) == 0


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_valid_calls_fail_loudly_without_a_gpu(lib):
    assert lib.tb200_kv4_append(C.byref(rows_args()), None) != 0
    assert lib.tb200_kv4_read(C.byref(rows_args()), None) != 0
    assert lib.tb200_attn_window(C.byref(attn_args()), None) != 0
    assert lib.tb200_kv4_attn(C.byref(attn_args()), None) != 0


def test_struct_layout(tmp_path):
    src = tmp_path / "sz.c"
    fields = [("tb200_kv4_rows_args", L.Kv4RowsArgs), ("tb200_cache_attn_args", L.CacheAttnArgs)]
    names = [(s, f) for s, c in fields for f, _ in c._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "trinity_b200.h"\nint main(){'
                   + "".join(f'printf("%zu ", offsetof({s},{f}));' for s, f in names)
                   + "".join(f'printf("%zu ", sizeof({s}));' for s, _ in fields) + "}")
    exe = tmp_path / "sz"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = [int(v) for v in subprocess.check_output([str(exe)]).split()]
    assert got == [getattr(c, f).offset for _, c in fields for f, _ in c._fields_] + [C.sizeof(c) for _, c in fields]


def test_python_wrappers_refuse_cpu_tensors(lib):
    from trinity_b200 import ops
    cache = ops.kv4_cache(1, 1, 6, 64, torch.float16, "cpu")
    assert cache.k_codes.shape == (1, 1, 8, 32) and cache.v_meta.shape == (1, 1, 8, 1, 2)
    x = torch.zeros(1, 1, 2, 64, dtype=torch.float16)
    lens = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.kv4_append(cache, x, x, 0), lambda: ops.kv4_read(cache, 0, 2), lambda: ops.kv4_attn(x, cache, lens),
                 lambda: ops.attn_window(x, x, x, lens)):
        with pytest.raises(ValueError, match="CUDA tensors"):
            call()
    with pytest.raises(ValueError):
        ops.kv4_cache(1, 1, 4, 96, torch.float16, "cpu")
