"""Ranges of the arguments of attention over caches (no GPU)."""
import ctypes as C

import pytest
import torch

from tests.test_cache_attn_checks import INVALID, attn_args, lib  # noqa: F401  (a fixture)


@pytest.mark.parametrize("scale,status", [(1e-30, 0), (0.9e-30, INVALID), (1e38, 0), (1.1e38, INVALID)])
def test_scale(lib, scale, status):  # noqa: F811
    for name in ("tb200_attn_window", "tb200_kv4_attn"):
        # (1e-30 and 1e38 as floats)
        assert getattr(lib, name + "_check")(C.byref(attn_args(sm_scale=float(torch.tensor(scale, dtype=torch.float32))))) == status
