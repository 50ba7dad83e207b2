"""The operators around a key-value cache where ordinary inputs do not lead: infinite values, weights far below the
largest, padding under weights that are no numbers, reports next to one another, units of several heads."""
import math
import subprocess
import sys
import textwrap
from pathlib import Path

import pytest
import torch

import plain_heads as plain
from intent_b200 import _native, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16, I8, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn


def randn(*shape, dtype=F32, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# --------------------------------------------------------------------------------- attention
def one_sequence(k, v, group, dtype, store, page=16, room=0):
    """A cache that holds rows k, v (length, kv_heads, columns) of one sequence, its pages in falling order, and a table with
    `room` more columns than it needs."""
    length, kv_heads, columns = k.shape
    pages = -(-length // page)
    kc, vc, ks, vs = plain.new_cache(pages, kv_heads, page, columns, store, "tokens", DEV)
    order = torch.arange(pages - 1, -1, -1, device=DEV)
    slots = (order[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)[:length]
    ops.cache_write(k.to(dtype), v.to(dtype), slots, kc, vc, ks, vs)
    table = torch.cat((order, torch.full((room,), -1, device=DEV))).to(torch.int32)[None]
    return {"k_cache": kc, "v_cache": vc, "k_scale": ks, "v_scale": vs, "block_table": table, "lengths": int32([length])}


def attend(q, case, scale):
    out, lse = ops.paged_attention(q, case["k_cache"], case["v_cache"], case["block_table"], case["lengths"], scale,
                                   k_scale=case["k_scale"], v_scale=case["v_scale"], return_lse=True)
    ops.workspace_status(DEV)
    return out, lse


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [1, 4, 7, 16])
@pytest.mark.parametrize("length, room", [(1, 0), (70, 0), (1500, 0), (5000, 300)])
def test_an_infinite_value_gives_that_infinity(length, room, group, dtype):
    """Whatever its weight is, and however it is rounded; two of both signs give NaN, and so does one under a key whose
    score is -infinity.  Every other column is what it would be without them."""
    k, v = randn(length, 2, 64, seed=length), randn(length, 2, 64, seed=length + 1)
    q = (2 * randn(1, 2 * group, 64, seed=group)).to(dtype)
    inf, last = float("inf"), length - 1
    v[0, 0, 3], v[last, 0, 9], v[length // 2, 1, 20] = inf, -inf, inf
    v[length // 3, 1, 63], v[last, 1, 62] = float("nan"), -inf
    if length > 4:
        v[2, 0, 30], v[length - 3, 0, 30] = inf, -inf
        k[last, 1] = -300 * q[0, group].float()            # far below the others, but not -infinity
    case = one_sequence(k, v, group, dtype, dtype, room=room)
    out, lse = attend(q, case, 0.125)
    expected, slack, expected_lse, lse_slack = plain.attention(q, case["k_cache"], case["v_cache"], None, None, case["block_table"],
                                                               case["lengths"], 0.125)
    expected[0, group:, 20], expected[0, group:, 62] = inf, -inf      # a weight that 64 bits do not hold is a weight all the same
    assert (out[0, :group, 3] == inf).all() and (out[0, :group, 9] == -inf).all() and (out[0, group:, 20] == inf).all()
    plain.close(out, expected, slack)
    plain.close(lse, expected_lse, lse_slack)
    # a key of -infinity weighs nothing, and nothing times an infinity is no number
    if length > 4:
        q, k[length // 2, 1] = q.abs() + 0.1, -inf
        case = one_sequence(k, v, group, dtype, dtype, room=room)
        out, lse = attend(q, case, 0.125)
        assert out[0, group:, 20].isnan().all() and lse.isfinite().all() and (out[0, :group, 3] == inf).all()
        assert out[0, group:, :20].isfinite().all()
