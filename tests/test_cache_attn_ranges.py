"""Ranges of the arguments of attention over caches, and what an empty 4-bit cache may be (no GPU)."""
import ctypes as C

import pytest
import torch

from tests.test_cache_attn_checks import INVALID, attn_args, lib  # noqa: F401  (a fixture)
from trinity_b200 import ops


@pytest.mark.parametrize("scale,status", [(1e-30, 0), (0.9e-30, INVALID), (1e38, 0), (1.1e38, INVALID)])
def test_scale(lib, scale, status):  # noqa: F811
    for name in ("tb200_attn_window", "tb200_kv4_attn"):
        # (1e-30 and 1e38 as floats)
        assert getattr(lib, name + "_check")(C.byref(attn_args(sm_scale=float(torch.tensor(scale, dtype=torch.float32))))) == status


@pytest.mark.parametrize("head_dim", [0, 32, 192, 256, -64])
def test_a_cache_that_no_operator_takes_is_not_made(head_dim):
    with pytest.raises(ValueError, match="head_dim"):
        ops.kv4_cache(1, 1, 4, head_dim, torch.bfloat16, "cpu")


def test_types_and_lengths_of_a_cache():
    for dtype in (torch.float32, torch.uint8, torch.float64):
        with pytest.raises(TypeError):
            ops.kv4_cache(1, 1, 4, 64, dtype, "cpu")
    with pytest.raises(ValueError, match="cache_len"):
        ops.kv4_cache(1, 1, -3, 64, torch.float16, "cpu")     # (would round up to 0)
    assert [ops.kv4_cache(2, 1, n, 128, torch.float16, "cpu").v_meta.shape for n in (0, 1, 4)] == [(2, 1, m, 2, 2) for m in (0, 4, 4)]
