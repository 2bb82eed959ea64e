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


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("kv_dt,D", [(BF, 128), (F16, 64), (E4M3, 128), (BF, 256), (E4M3, 256)])
def test_one_token_that_does_not_see_itself(kv_dt, D, bad):
    """A request of one token whose mask hides the token's own row: whatever the row holds stays out,
    over a cache and over none."""
    if kv_dt == E4M3 and not math.isnan(bad):
        pytest.skip("e4m3 has no infinities")
    x = make([1, 70, 1300], [1, 1, 1], 4, 2, D, F16 if kv_dt == F16 else BF, kv_dt, 16, seed=D)
    for j, n in enumerate(x["lens"]):
        x["seen"][j][0] = False
        x["mask"][j] = 0
        page = int(x["table"][j, (n - 1) // 16])
        for name in ("k", "v"):
            pool = x[name].float()
            pool[page, (n - 1) % 16] = bad
            x[name] = pool.to(kv_dt)
    out, lse = call(x)
    assert bool((out[0] == 0).all()) and bool((lse[0] == -math.inf).all())
    ph.check_attn((out, lse), want(x))
    # a mask that shows the row again
    x["seen"][1][0] = True
    x["mask"][1] = 1
    out, lse = call(x)
    assert not torch.isfinite(out[1].float()).any()
    ph.check_attn((out, lse), want(x), torch.tensor([True, False, True]))
    assert_device_ok()
