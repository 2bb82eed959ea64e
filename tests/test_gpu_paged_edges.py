"""Edges of the paged-cache operators: partly filled warps, hidden rows, unaligned views, bounds that
run past the tensors."""

import math

import pytest
import torch

import paged_helpers as ph
from gpu_helpers import assert_device_ok
from test_gpu_paged_tree import call, dev, make, want

pytestmark = pytest.mark.gpu

BF, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("kv_dt", [BF, F16, E4M3])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 31, 33, 65, 97])
def test_partly_filled_warps(kv_dt, D, rows):
    """A row tile that ends inside a warp, whole and in parts: its rows, and only those, come out."""
    q_dt = F16 if kv_dt == F16 else BF
    x = make([90, rows + 3000], [rows, rows], 1, 1, D, q_dt, kv_dt, 32, seed=rows + D)
    ph.check_attn(call(x), want(x))
    assert_device_ok()
