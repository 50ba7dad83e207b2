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


@pytest.mark.parametrize("dtype, store", [(F16, F16), (BF16, BF16), (F16, I8), (BF16, E4M3)])
@pytest.mark.parametrize("group", [1, 4, 7, 16])
@pytest.mark.parametrize("length, room", [(450, 0), (4096, 0), (4096, 8000)])
def test_small_weights_behind_a_sink_count(length, room, group, dtype, store):
    """One key takes nearly all of the softmax and its value is zero but for one column, so the others are what all the other
    keys hold, each 24 to 32 powers of two below it.  A weight enters as two halves, the second 2^-11 of the first's steps: in f16 (the products of f16
    rows and of codes) that keeps what is above 2^-36, with the largest weight at 2^7 or more, so each is off
    by at most 2^-43 of the largest (times its row's scale over the largest product's), beside 2^-16 of itself."""
    scale = 1 / 16
    for below in (24.0, 26.0, 32.0):
        k, v = torch.zeros(length, 1, 128, device=DEV), randn(length, 1, 128, seed=3) + 0.5
        k[:, 0, 0] = -(below + 1.0 * (torch.rand(length, generator=torch.Generator().manual_seed(int(below))).to(DEV) - 0.5)) * math.log(2.0)
        k[1, 0, 0], v[1] = 0.0, 0.0
        v[1, 0, 0] = 1.0
        q = torch.zeros(1, group, 128, device=DEV)
        q[..., 0] = 1 / scale
        q = q.to(dtype)
        case = one_sequence(k, v, group, dtype, store, room=room)
        out, lse = attend(q, case, scale)
        rows = []
        for cache, size in ((case["k_cache"], case["k_scale"]), (case["v_cache"], case["v_scale"])):
            wide = plain.values(cache, size)[case["block_table"][0, :-(-length // 16)].long()]
            rows.append(wide.permute(1, 0, 2, 3).reshape(-1, 128)[:length])
        scores = rows[0] @ q[0, 0].double() * scale
        weights = torch.softmax(scores, 0)
        sizes = torch.ones(length, dtype=torch.float64, device=DEV)
        if case["v_scale"] is not None:
            sizes = case["v_scale"][case["block_table"][0, :-(-length // 16)].long()].double().reshape(-1)[:length]
        expected = (weights[:, None] * rows[1]).sum(0)
        # a score of magnitude 33 is rounded once from its product and once when scaled (2^-24 each, of 33 log2 e), and the
        # difference to the base once more; exp2 and log2 add 2^-20
        delta = 4 * 48 * plain.F32 + 2.0 ** -20
        size = (weights[:, None] * rows[1].abs()).sum(0)
        slack = (2 * delta + 2.0 ** -16 + (length / 64 + 64) * plain.F32) * size
        if store != BF16:
            slack = slack + 2.0 ** -43 * (weights * sizes).amax() * (rows[1].abs() / sizes[:, None]).sum(0)
        plain.close(out, expected.expand(1, group, 128), slack)
        plain.close(lse, torch.logsumexp(scores, 0).expand(1, group), delta + (length / 64 + 64) * plain.F32)


@pytest.mark.parametrize("group", [1, 7, 16])
@pytest.mark.parametrize("length, room", [(200, 0), (3000, 0)])
def test_values_near_the_end_of_bf16(length, room, group):
    """The largest numbers of bf16, under scores that rise slowly: a weight is at most 1, whatever the base was when it came."""
    k, v = torch.zeros(length, 1, 64, device=DEV), torch.zeros(length, 1, 64, device=DEV)
    k[:, 0, 0] = torch.linspace(0, 5, length, device=DEV)             # 7.2 in units of log2: the base does not follow
    v[length - 2, 0, :32], v[length - 1, 0, 32:], v[0, 0, 5] = -3.3e38, 3.3e38, 3e38
    q = torch.zeros(1, group, 64, device=DEV, dtype=BF16)
    q[..., 0] = 1
    case = one_sequence(k, v, group, BF16, BF16, room=room)
    out, lse = attend(q, case, 1.0)
    expected, slack, expected_lse, lse_slack = plain.attention(q, case["k_cache"], case["v_cache"], None, None, case["block_table"],
                                                               case["lengths"], 1.0)
    plain.close(out, expected, slack)
    plain.close(lse, expected_lse, lse_slack)


def test_a_table_without_columns_has_lost_what_a_sequence_holds():
    q = randn(3, 4, 64, dtype=F16)
    case = one_sequence(randn(20, 2, 64), randn(20, 2, 64), 2, F16, F16)
    out, lse = ops.paged_attention(q, case["k_cache"], case["v_cache"], case["block_table"].expand(3, -1)[:, :0], int32([0, 5, -3]), 0.125,
                                   return_lse=True)
    with pytest.raises(ValueError, match=r"\(row 1\)"):
        ops.workspace_status(DEV)
    assert not out[0].any() and not out[2].any() and out[1].isnan().all() and (lse == -float("inf")).all()


# ------------------------------------------------------------------------ norm and rotation
def rotary_inputs(tokens, heads, kv_heads, columns, pairs, dtype, seed=0):
    both = randn(tokens, heads + kv_heads + 1, columns, dtype=dtype, seed=seed)
    w = (1 + 0.3 * randn(2, columns, seed=seed + 1)).to(dtype)
    angle = torch.rand(64, pairs, device=DEV, dtype=torch.float64, generator=torch.Generator(device=DEV).manual_seed(seed)) * 7
    positions = torch.arange(tokens, device=DEV, dtype=torch.int32) * 7 % 64
    return both[:, :heads], both[:, heads:heads + kv_heads], w[0], w[1], angle.cos().float(), angle.sin().float(), positions


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_padding_gets_zero_gradients_under_any_weight(dtype):
    q, k, qw, kw, cos, sin, positions = rotary_inputs(40, 4, 2, 64, 16, dtype, seed=3)
    clean = ops.head_norm_rotary_backward(q, k, q, k, qw, kw, cos, sin, positions)
    positions[::3] = -1
    positions[31] = 64
    qw[5], qw[40], kw[20] = float("inf"), float("nan"), -float("inf")
    grads = ops.head_norm_rotary_backward(q, k, q, k, qw, kw, cos, sin, positions)
    with pytest.raises(ValueError, match=r"\(row 31\)"):
        ops.workspace_status(DEV)
    absent = (positions < 0) | (positions > 63)
    assert not grads[0][absent].any() and not grads[1][absent].any()
    assert grads[0][~absent].isnan().all() and clean[0].isfinite().all()
    # the weights' gradients do not depend on the weights
    for i, (g, x, w) in enumerate(((q, q, qw), (k, k, kw))):
        _, _, dw, dw_slack = plain.norm_rotary_backward(g, x, torch.ones_like(w), cos, sin, positions, 1e-6, False)
        plain.close(grads[2 + i], dw, dw_slack)


# ----------------------------------------------------------------------------------- the call
def test_an_output_that_does_not_fit_raises_torchs_error():
    """275 GB of rows: what catches torch.OutOfMemoryError to make room catches this."""
    cache = torch.zeros(1, 64, 1, 128, dtype=F16, device=DEV)
    slots = torch.zeros(1, dtype=torch.int64, device=DEV).expand(1 << 24)
    with pytest.raises(torch.OutOfMemoryError):
        ops.cache_read(cache, cache, slots)
    back = ops.cache_read(cache, cache, slots[:3])
    assert back[0].shape == (3, 64, 128) and not back[0].any()


def test_a_bad_index_does_not_hide_a_wait_that_gave_up():
    cache = torch.zeros(1, 1, 16, 64, dtype=F16, device=DEV)
    rows, far = randn(2, 1, 64, dtype=F16), torch.tensor([1, 99], device=DEV)

    def bad_slot():
        ops.cache_write(rows, rows, far, cache, cache.clone())

    def wait_that_gives_up():
        space = ops.workspace(DEV)
        status = _native.entry("b200_selftest_bounded_wait")(space.data_ptr(), space.numel(), 1, 100_000, torch.cuda.current_stream().cuda_stream)
        _native.check("b200_selftest_bounded_wait", status)

    for first, second in ((bad_slot, wait_that_gives_up), (wait_that_gives_up, bad_slot)):
        first()
        second()
        with pytest.raises(_native.NativeCallError) as error:
            ops.workspace_status(DEV)
        assert error.value.status == _native.ERR_DEVICE_TIMEOUT
        ops.workspace_status(DEV)
    bad_slot()
    with pytest.raises(ValueError, match=r"\(row 1\)"):
        ops.workspace_status(DEV)
    ops.workspace_status(DEV)


@pytest.mark.parametrize("first", ["c = ops.gemm(a, b)", "ops.cache_write(rows, rows, good, cache, other); c = ops.gemm(a, b)"])
def test_a_first_call_inside_a_capture_leaves_later_reports_alone(first):
    """In a process of its own: the first call on the device is a captured one, so its status words must neither come
    from the graph's memory nor be cleared by its replays."""
    program = textwrap.dedent("""
        import torch
        from intent_b200 import ops
        a = torch.randn(256, 256, device="cuda:0").bfloat16()
        b = a.t()
        cache = torch.zeros(1, 1, 16, 64, device="cuda:0").half()
        rows, other = torch.ones(2, 1, 64, device="cuda:0").half(), cache.clone()
        good, bad = torch.tensor([1, 5], device="cuda:0"), torch.tensor([1, 99], device="cuda:0")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            FIRST
            out = ops.softmax(c)
        ops.workspace_status("cuda:0")                      # nothing has run: nothing to report
        ops.cache_write(rows, rows, bad, cache, other)
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        try:
            ops.workspace_status("cuda:0")
        except ValueError as error:
            assert "row 1" in str(error), error
        else:
            raise SystemExit("the replays cleared the report")
        ops.workspace_status("cuda:0")
        want = a.double() @ b.double()
        assert (c.double() - want).abs().max() <= 2.0 ** -8 * want.abs().max()
        cache.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert int((cache[0, 0, :, 0] == 1).sum()) == (2 if "cache_write" in 'FIRST' else 0)
        del graph
        print("held")
    """).replace("FIRST", first)
    done = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=600, cwd=Path(__file__).resolve().parents[1])
    assert done.returncode == 0 and "held" in done.stdout, done.stdout + done.stderr


def unit_rows(tokens, heads, kv_heads, columns):
    """Heads of a token that one group of lanes takes, by the rule beside the kernel (rotary.cu, rows_of_unit)."""
    lanes = 1
    while lanes * 16 < columns:
        lanes *= 2
    groups = 2 * torch.cuda.get_device_properties(0).multi_processor_count * 256 // lanes
    for rows in range(8, 1, -1):
        units = -(-heads // rows) + -(-kv_heads // rows)
        if tokens * units >= groups and units * rows * 7 <= (heads + kv_heads) * 8:
            return rows
    return 1


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens, heads, kv_heads, columns, pairs, rows", [
    (6500, 5, 3, 64, 32, 3),           # 5 = 3 + 2: a unit that is not full
    (9600, 7, 7, 64, 16, 8), (2400, 32, 8, 128, 64, 8), (2500, 31, 8, 128, 32, 8), (3300, 13, 2, 256, 128, 2), (19000, 15, 2, 48, 24, 3)])
def test_units_of_several_heads(tokens, heads, kv_heads, columns, pairs, rows, interleaved, dtype):
    """Calls large enough that a group of lanes takes several heads of a token, and not always as many; padding, rows of zeros
    and an epsilon of 0, so that a row that is not there would show."""
    assert unit_rows(tokens, heads, kv_heads, columns) == rows
    q, k, qw, kw, cos, sin, positions = rotary_inputs(tokens, heads, kv_heads, columns, pairs, dtype, seed=tokens)
    q, k = q.clone(), k.clone()
    positions[::7] = -1
    q[::7], k[::7] = 0, float("nan")
    live = (positions >= 0)[:, None, None]
    out = ops.head_norm_rotary(q, k, qw, kw, cos, sin, positions, 0.0, interleaved=interleaved)
    gq, gk = randn(*q.shape, dtype=dtype, seed=71), randn(*k.shape, dtype=dtype, seed=72)
    grads = ops.head_norm_rotary_backward(gq, gk, q, k, qw, kw, cos, sin, positions, 0.0, interleaved=interleaved)
    ops.workspace_status(DEV)
    for i, (x, w, g) in enumerate(((q, qw, gq), (k, kw, gk))):
        x = torch.where(live, x, 1.0)
        plain.close(out[i], *plain.norm_rotary(x, w, cos, sin, positions, 0.0, interleaved))
        dx, dx_slack, dw, dw_slack = plain.norm_rotary_backward(g, x, w, cos, sin, positions, 0.0, interleaved)
        plain.close(grads[i], dx, dx_slack)
        # no lane adds more than 256 rows here either
        plain.close(grads[2 + i], dw, dw_slack)
    in_place = ops.head_norm_rotary_backward(gq, gk, q, k, qw, kw, cos, sin, positions, 0.0, interleaved=interleaved, dq=gq, dk=gk)
    assert all(torch.equal(a, b) for a, b in zip(in_place, grads))
    in_place = ops.head_norm_rotary(q, k, qw, kw, cos, sin, positions, 0.0, interleaved=interleaved, q_out=q, k_out=k)
    assert all(torch.equal(a, b) for a, b in zip(in_place, out))


@pytest.mark.parametrize("dtype, store", [(F16, F16), (BF16, BF16), (F16, I8), (BF16, E4M3)])
@pytest.mark.parametrize("group", [4, 7, 16])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 14, 2.0 ** 15.4])
def test_equal_values_come_back_whatever_the_scores(size, group, dtype, store):
    """Scores of up to 2^34, of which f32 holds no fraction: weights add up to 1 all the same, so the result is the value.  A
    weight is off by 2^-16 of itself at most, its sums by 2^-24 for each of their terms."""
    for length, room in ((300, 0), (3000, 0)):
        k = size * (1 + torch.rand(length, 1, 64, generator=torch.Generator().manual_seed(length)).to(DEV))
        q = (size * (1 + torch.rand(1, group, 64, generator=torch.Generator().manual_seed(group)).to(DEV))).clamp(max=60000).to(dtype)
        for sign in (1.0, -1.0):
            case = one_sequence(sign * k.clamp(max=60000), torch.ones(length, 1, 64, device=DEV), group, dtype, store, room=room)
            out, lse = attend(q, case, 0.5)
            value = plain.values(case["v_cache"], case["v_scale"])[case["block_table"][0, 0].long(), 0, 0, 0]
            plain.close(out, value.expand(1, group, 64), 2.0 ** -15 + (length + 64) * plain.F32)
            assert lse.isfinite().all()


def test_a_first_call_in_inference_mode_leaves_reports_readable_outside():
    """In a process of its own: status words made in inference mode could not be cleared outside of it."""
    program = textwrap.dedent("""
        import torch
        from intent_b200 import ops
        cache = torch.zeros(1, 1, 16, 64, device="cuda:0").half()
        rows, bad = torch.ones(2, 1, 64, device="cuda:0").half(), torch.tensor([1, 99], device="cuda:0")
        with torch.inference_mode():
            ops.cache_write(rows, rows, bad, cache, cache.clone())
        for expected in (True, False):
            try:
                ops.workspace_status("cuda:0")
                reported = False
            except ValueError as error:
                reported = "row 1" in str(error)
            assert reported == expected
        print("held")
    """)
    done = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=600, cwd=Path(__file__).resolve().parents[1])
    assert done.returncode == 0 and "held" in done.stdout, done.stdout + done.stderr
