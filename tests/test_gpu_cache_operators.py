"""The operators around a key-value cache on a device, against their plain forms in 64 bits
(plain_heads, whose bounds come from the inputs): per-head norm with rotation and its gradient, writing and
reading a paged cache in 16 and 8 bits, attention of one new token over it, and all of them in a row."""
import pytest
import torch

import plain_heads as plain
from intent_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16, I8, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn


def randn(*shape, dtype=F32, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def no_status():
    ops.workspace_status(DEV)


def status_names(row):
    """A kernel reported `row`, and the report is cleared by reading it."""
    with pytest.raises(ValueError, match=rf"outside its table or cache \(row {row}\)"):
        ops.workspace_status(DEV)
    ops.workspace_status(DEV)


# ------------------------------------------------------------------------ norm and rotation
def rotary_inputs(tokens, heads, kv_heads, columns, pairs, dtype, seed=0):
    both = randn(tokens, heads + kv_heads + 1, columns, dtype=dtype, seed=seed)
    w = (1 + 0.3 * randn(2, columns, seed=seed + 1)).to(dtype)
    angle = torch.rand(64, pairs, device=DEV, dtype=torch.float64, generator=torch.Generator(device=DEV).manual_seed(seed)) * 7
    positions = torch.arange(tokens, device=DEV, dtype=torch.int32) * 7 % 64
    return both[:, :heads], both[:, heads:heads + kv_heads], w[0], w[1], angle.cos().float(), angle.sin().float(), positions


ROTARY = [  # tokens, heads, kv_heads, columns, pairs
    (1, 1, 1, 16, 8), (1, 32, 8, 128, 64), (3, 5, 1, 32, 16), (37, 4, 4, 64, 32), (130, 12, 3, 80, 40), (33, 6, 2, 96, 16),
    (65, 9, 2, 128, 64), (19, 7, 7, 256, 128), (21, 3, 2, 208, 72), (300, 33, 9, 64, 8), (513, 32, 8, 128, 64)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens, heads, kv_heads, columns, pairs", ROTARY)
def test_head_norm_rotary(tokens, heads, kv_heads, columns, pairs, interleaved, dtype):
    q, k, qw, kw, cos, sin, positions = rotary_inputs(tokens, heads, kv_heads, columns, pairs, dtype, seed=tokens)
    if tokens > 2:
        positions[tokens // 2] = -1
    q_out, k_out = ops.head_norm_rotary(q, k, qw, kw, cos, sin, positions, 1e-5, interleaved=interleaved)
    no_status()
    for out, x, w in ((q_out, q, qw), (k_out, k, kw)):
        plain.close(out, *plain.norm_rotary(x, w, cos, sin, positions, 1e-5, interleaved))
        if tokens > 2:
            assert not out[tokens // 2].any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens, heads, kv_heads, columns, pairs", ROTARY)
def test_head_norm_rotary_backward(tokens, heads, kv_heads, columns, pairs, interleaved, dtype):
    q, k, qw, kw, cos, sin, positions = rotary_inputs(tokens, heads, kv_heads, columns, pairs, dtype, seed=tokens)
    if tokens > 2:
        positions[tokens // 2] = -1
    gq, gk = randn(*q.shape, dtype=dtype, seed=71), randn(*k.shape, dtype=dtype, seed=72)
    result = ops.head_norm_rotary_backward(gq, gk, q, k, qw, kw, cos, sin, positions, 1e-5, interleaved=interleaved)
    no_status()
    for i, (g, x, w) in enumerate(((gq, q, qw), (gk, k, kw))):
        dx, dx_slack, dw, dw_slack = plain.norm_rotary_backward(g, x, w, cos, sin, positions, 1e-5, interleaved)
        plain.close(result[i], dx, dx_slack)
        plain.close(result[2 + i], dw, dw_slack)
    again = ops.head_norm_rotary_backward(gq, gk, q, k, qw, kw, cos, sin, positions, 1e-5, interleaved=interleaved)
    assert all(torch.equal(a, b) for a, b in zip(result, again))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient_against_differences(interleaved):
    """The slope of the kernel's own forward pass in f32 along a direction, by central differences.
    With h = 2^-6 the difference's third-order term is below h^2 times the slope's size, and rounding adds
    32 half steps of each |y| |g| over h (the same bound that the forward test uses)."""
    q, k, qw, kw, cos, sin, positions = rotary_inputs(40, 6, 2, 64, 16, F32, seed=5)
    q, k = q.contiguous(), k.contiguous()
    gq, gk, sq, sk, sw = randn(*q.shape, seed=6), randn(*k.shape, seed=7), randn(*q.shape, seed=8), randn(*k.shape, seed=9), randn(64, seed=10)

    def loss(h):
        yq, yk = ops.head_norm_rotary(q + h * sq, k + h * sk, qw + h * sw, kw + h * sw, cos, sin, positions, 1e-5, interleaved=interleaved)
        size = (yq.abs().amax(-1, keepdim=True) * gq).double().abs().sum() + (yk.abs().amax(-1, keepdim=True) * gk).double().abs().sum()
        return (yq.double() * gq).sum() + (yk.double() * gk).sum(), size

    h = 2.0 ** -6
    dq, dk, dqw, dkw = ops.head_norm_rotary_backward(gq, gk, q, k, qw, kw, cos, sin, positions, 1e-5, interleaved=interleaved)
    parts = ((dq.double() * sq), (dk.double() * sk), (dqw.double() * sw), (dkw.double() * sw))
    (up, size), (down, _) = loss(h), loss(-h)
    bound = 32 * plain.F32 * size / h + 8 * h * h * sum(p.abs().sum() for p in parts)
    assert abs((up - down) / (2 * h) - sum(p.sum() for p in parts)) <= bound


def test_rotary_in_place_in_a_fused_tensor():
    for backward in (False, True):
        q, k, qw, kw, cos, sin, positions = rotary_inputs(50, 8, 2, 128, 64, BF16, seed=3)
        rest = q.as_strided(q._base.shape, q._base.stride())[:, 10:]
        before, kept = [t.clone() for t in (q, k)], rest.clone()
        if backward:
            gq, gk = randn(*q.shape, dtype=BF16, seed=4), randn(*k.shape, dtype=BF16, seed=5)
            expected = ops.head_norm_rotary_backward(gq, gk, *before, qw, kw, cos, sin, positions)
            got = ops.head_norm_rotary_backward(gq, gk, q, k, qw, kw, cos, sin, positions, dq=q, dk=gk)
        else:
            expected = ops.head_norm_rotary(*before, qw, kw, cos, sin, positions)
            got = ops.head_norm_rotary(q, k, qw, kw, cos, sin, positions, q_out=q, k_out=k)
        assert all(torch.equal(a, b) for a, b in zip(got, expected)) and torch.equal(rest, kept)


def test_rotary_edges():
    q, k, qw, kw, cos, sin, positions = rotary_inputs(9, 2, 1, 64, 16, F32, seed=6)
    q, k = q.clone(), k.clone()
    q[1] = 0                                         # a row of zeros stays zeros
    q[2, 0, 40], q[3, 1, 50], q[4, 0, 3] = float("inf"), float("nan"), float("inf")
    q[5, :, :] = float("nan")
    positions[5] = -7                                # padding hides what it holds
    positions[7] = 64                                # one row behind the tables
    q_out, k_out = ops.head_norm_rotary(q, k, qw, kw, cos, sin, positions)
    status_names(7)
    live = positions < 64
    expected, _ = plain.norm_rotary(q, qw, cos, sin, positions, 1e-6, False)
    assert not q_out[1].any() and not q_out[5].any() and not q_out[7].any() and not k_out[7].any()
    assert torch.equal(q_out.isnan(), expected.isnan())
    assert q_out[2, 0].isnan().sum() == 1            # an infinity in a column that passes spoils itself alone
    assert q_out[3, 1].isnan().all() and q_out[4, 0].isnan().sum() == 2
    plain.close(k_out[live], *(t[live] for t in plain.norm_rotary(k, kw, cos, sin, positions, 1e-6, False)))
    grads = ops.head_norm_rotary_backward(q_out, k_out, q, k, qw, kw, cos, sin, positions)
    status_names(7)
    assert not grads[0][5].any() and not grads[0][7].any() and not grads[1][7].any()
    # nothing to do
    none = ops.head_norm_rotary_backward(q[:0], k[:0], q[:0], k[:0], qw, kw, cos, sin, positions[:0])
    assert none[0].shape == (0, 2, 64) and not none[2].any() and not none[3].any()
    only_q = ops.head_norm_rotary_backward(k_out, k_out[:, :0], k, k[:, :0], qw, kw, cos, sin, positions)
    assert not only_q[3].any() and only_q[1].shape == (9, 0, 64)
    status_names(7)
    # padding and heads that fill no whole unit add nothing even where a row of zeros has no norm
    many = [randn(3000, n, 64, seed=n) for n in (5, 3, 5, 3)]
    places = torch.arange(3000, device=DEV, dtype=torch.int32) % 64
    places[::7] = -1
    for t in many:
        t[::7] = 0
    grads = ops.head_norm_rotary_backward(*many, qw, kw, cos, sin, places, 0.0)
    for i in range(2):
        dx, dx_slack, dw, dw_slack = plain.norm_rotary_backward(many[i], torch.where(places[:, None, None] < 0, 1.0, many[2 + i]),
                                                                (qw, kw)[i], cos, sin, places, 0.0, False)
        plain.close(grads[i], dx, dx_slack)
        plain.close(grads[2 + i], dw, dw_slack)
    with pytest.raises(TypeError):
        ops.head_norm_rotary(q, k, qw, kw, cos, sin, positions.long())
    with pytest.raises(NotImplementedError):
        ops.head_norm_rotary(q[..., :40], k[..., :40], qw[:40], kw[:40], cos, sin, positions)
    with pytest.raises(ValueError):
        ops.head_norm_rotary(q, k, qw, kw, cos, sin, positions, q_out=k)


def test_rotary_strides_and_nothing():
    """Positions, tables and heads that repeat (stride 0) or skip; no tokens; one output given."""
    q, k, qw, kw, cos, sin, positions = rotary_inputs(12, 4, 4, 64, 32, F16, seed=9)
    one = int32([17]).expand(12)
    apart = torch.stack((positions, positions + 1), 1)[:, 0]
    for places in (one, apart):
        got = ops.head_norm_rotary(q[::2], k[::2], qw, kw, cos, sin, places[::2], 1e-5, k_out=torch.empty(6, 4, 64, dtype=F16, device=DEV))
        for out, x, w in zip(got, (q[::2], k[::2]), (qw, kw)):
            plain.close(out, *plain.norm_rotary(x, w, cos, sin, places[::2], 1e-5, False))
    shared = k[:, :1].expand(12, 4, 64)
    flat = cos[3:4].expand(64, 32), sin[3:4].expand(64, 32)
    got = ops.head_norm_rotary(q, shared, qw, kw, *flat, positions, 1e-5)
    plain.close(got[1], *plain.norm_rotary(shared, kw, *flat, positions, 1e-5, False))
    assert ops.head_norm_rotary(q[:0], k[:0], qw, kw, cos, sin, positions[:0])[1].shape == (0, 4, 64)
    assert ops.head_norm_rotary(q[:, :0], k, qw, kw, cos, sin, positions)[0].shape == (12, 0, 64)
    with pytest.raises(ValueError):
        ops.head_norm_rotary(q, k, qw, kw, cos, sin, positions, q_out=k)          # the other's input
    with pytest.raises(ValueError):
        ops.head_norm_rotary(q, shared, qw, kw, cos, sin, positions, k_out=shared)
    no_status()


# --------------------------------------------------------------------------------- the cache
def cache_rows(tokens, heads, columns, dtype, seed=0):
    both = randn(tokens, 2 * heads + 1, columns, dtype=F32, seed=seed) * torch.exp(1.5 * randn(tokens, 2 * heads + 1, 1, seed=seed + 1))
    both = both.to(dtype)
    return both[:, :heads], both[:, heads:2 * heads]


CACHE = [  # tokens, heads, columns, page, pages, layout
    (1, 1, 16, 1, 1, "heads"), (1, 8, 128, 16, 3, "tokens"), (5, 3, 64, 7, 4, "apart"), (77, 2, 96, 16, 6, "heads"),
    (200, 4, 128, 100, 3, "tokens"), (130, 5, 256, 64, 4, "apart"), (33, 2, 80, 8, 9, "tokens"), (1000, 8, 128, 16, 70, "heads")]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("store", [None, I8, E4M3])
@pytest.mark.parametrize("tokens, heads, columns, page, pages, layout", CACHE)
def test_cache_write_and_read(tokens, heads, columns, page, pages, layout, store, dtype):
    store = store or dtype
    k, v = cache_rows(tokens, heads, columns, dtype, seed=tokens)
    kc, vc, ks, vs = plain.new_cache(pages, heads, page, columns, store, layout, DEV)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(tokens))[:tokens].to(DEV)
    if tokens > 3:
        slots[1] = -1
    bits = [None if t is None else t.clone().view({1: torch.int8, 2: torch.int16, 4: torch.int32}[t.element_size()]) for t in (kc, vc, ks, vs)]
    ops.cache_write(k, v, slots, kc, vc, ks, vs)
    no_status()
    live = (slots >= 0).nonzero().flatten()
    at, place = slots[live] // page, slots[live] % page
    for x, cache, scale in ((k, kc, ks), (v, vc, vs)):
        expected, expected_scale = (x.double(), None) if scale is None else plain.quantise(x, store)
        assert torch.equal(plain.values(cache, scale)[at, :, place], expected[live])
        if scale is not None:
            assert torch.equal(scale[at, :, place].double(), expected_scale[live])
    untouched = torch.ones((pages, page), dtype=torch.bool, device=DEV)
    untouched[at, place] = False
    for old, new in zip(bits, (kc, vc, ks, vs)):
        if old is not None:
            assert torch.equal(old.transpose(1, 2)[untouched], new.view(old.dtype).transpose(1, 2)[untouched])
    for out_dtype in ((dtype,) if store == dtype else (F16, BF16)):
        back = ops.cache_read(kc, vc, slots, ks, vs, dtype=out_dtype)
        no_status()
        for x, y in zip((k, v), back):
            exact = x.double() if store == dtype else plain.quantise(x, store)[0]
            rounded = exact.float().to(out_dtype)
            assert torch.equal(y[live], rounded[live]) and (tokens <= 3 or not y[1].any())


@pytest.mark.parametrize("store", [I8, E4M3])
def test_quantisation_at_its_borders(store):
    """Ties, values next to ties, subnormals, zeros, the largest numbers, infinities and NaN."""
    rows = torch.zeros(64, 1, 32)
    g = torch.Generator().manual_seed(1)
    for r in range(64):
        unit = 2.0 ** (r % 14 - 12)
        if r % 4 == 0:      # scale = unit exactly: every half is a tie
            rows[r, 0] = (torch.randint(-126, 126, (32,), generator=g) + 0.5) * unit
            rows[r, 0, 0] = 127 * unit
        elif r % 4 == 1:    # between e4m3's codes
            rows[r, 0] = torch.randint(-126, 127, (32,), generator=g) * unit
            rows[r, 0, 0] = (448 if r % 8 == 1 else 449) * unit * 2.0 ** -2
        elif r % 4 == 2:    # any scale, values around its halves
            top = 1 + torch.rand(1, generator=g)
            rows[r, 0] = (torch.randint(-126, 126, (32,), generator=g) + 0.5) * (top / 127) * unit
            rows[r, 0, 5] = top * unit
        else:
            rows[r, 0] = torch.randn(32, generator=g) * 2.0 ** -(r // 2)
    rows[3], rows[7, 0, :4], rows[11] = 0, 65504, rows[11] * 2.0 ** -130
    rows[15, 0, 3], rows[19, 0, 4], rows[23, 0, 9] = float("inf"), float("nan"), -float("inf")
    for dtype in (F16, BF16):
        x = rows.to(dtype).to(DEV)
        x = torch.where(x.isinf() & ~rows.to(DEV).isinf(), torch.zeros_like(x), x)
        kc, vc, ks, vs = plain.new_cache(8, 1, 8, 32, store, "apart", DEV)
        slots = torch.arange(64, device=DEV)
        ops.cache_write(x, -x, slots, kc, vc, ks, vs)
        expected, scale = plain.quantise(x, store)
        got_k, got_v = (plain.values(c, s).transpose(1, 2).reshape(64, 1, 32) for c, s in ((kc, ks), (vc, vs)))
        assert torch.equal(got_k.nan_to_num(7e77), expected.nan_to_num(7e77))
        assert torch.equal(got_v.nan_to_num(7e77), (-expected).nan_to_num(7e77))
        assert got_k[15].isnan().all() and got_k[19].isnan().all() and got_k[23].isnan().all()
        assert torch.equal(ks.transpose(1, 2).reshape(64, 1).double().nan_to_num(-1), scale.nan_to_num(-1))
        back, _ = ops.cache_read(kc, vc, slots, ks, vs, dtype=dtype)
        assert torch.equal(back.double().nan_to_num(7e77), expected.float().to(dtype).double().nan_to_num(7e77))


@pytest.mark.parametrize("store", [BF16, I8])
def test_slots_outside_the_cache_are_left_out_and_reported(store):
    k, v = cache_rows(6, 2, 64, BF16)
    kc, vc, ks, vs = plain.new_cache(2, 2, 4, 64, store, "heads", DEV)
    slots = torch.tensor([7, -1, 0, 8, 3, -(1 << 40)], device=DEV)
    ops.cache_write(k, v, slots, kc, vc, ks, vs)
    status_names(3)
    written = plain.values(kc, ks)[..., 0].isfinite().nonzero()
    assert {(p * 4 + s) for p, _, s in written.tolist()} == {0, 3, 7}
    far = slots.clone()
    far[3] = 1 << 40
    back = ops.cache_read(kc, vc, far, ks, vs, dtype=BF16)
    status_names(3)
    assert not back[0][[1, 3, 5]].any() and back[0][[0, 2, 4]].any()
    twice = ops.cache_read(kc, vc, torch.tensor([3, 3, 0, 3], device=DEV), ks, vs, dtype=BF16)     # reading a slot twice is fine
    assert torch.equal(twice[0][0], twice[0][3]) and torch.equal(twice[0][2], back[0][2])
    empty = [None if t is None else t[:0] for t in (kc, vc, ks, vs)]                 # a cache of no pages holds no slot
    ops.cache_write(k, v, slots, *empty)
    status_names("[0234]")                                                            # any of the four that name one
    nothing = ops.cache_read(kc, vc, slots[:0], ks, vs)
    assert nothing[0].shape == (0, 2, 64)
    ops.cache_write(k[:0], v[:0], slots[:0], kc, vc, ks, vs)
    no_status()


# --------------------------------------------------------------------------------- attention
def attention_case(lengths, kv_heads, group, columns, page, dtype, store, layout, seed=0, spread=1.0, table_order=None, slack_columns=1):
    batch, longest = len(lengths), max(max(lengths), 1)
    width = -(-longest // page) + slack_columns
    held = [-(-max(n, 0) // page) for n in lengths]
    pages = sum(held) + 2
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((batch, width), -1, dtype=torch.int32)
    kc, vc, ks, vs = plain.new_cache(pages, kv_heads, page, columns, store, layout, DEV)
    for b, n in enumerate(lengths):
        mine = [order.pop() for _ in range(held[b])]
        table[b, :held[b]] = torch.tensor(mine, dtype=torch.int32)
        if n <= 0:
            continue
        slots = (torch.tensor(mine)[:, None] * page + torch.arange(page)).reshape(-1)[:n].to(DEV)
        k = randn(n, kv_heads, columns, dtype=dtype, seed=seed * 1000 + 2 * b)
        v = randn(n, kv_heads, columns, seed=seed * 1000 + 2 * b + 1)
        v = (v * torch.exp(0.5 * randn(n, kv_heads, 1, seed=seed * 1000 + 3 * b))).to(dtype)
        ops.cache_write(k, v, slots, kc, vc, ks, vs)
    q = spread * randn(batch, kv_heads * group, columns, seed=seed + 17)
    return {"q": q.to(dtype), "k_cache": kc, "v_cache": vc, "block_table": table.to(DEV), "lengths": int32(lengths),
            "scale": columns ** -0.5, "k_scale": ks, "v_scale": vs}


def attend(case, **more):
    return ops.paged_attention(case["q"], case["k_cache"], case["v_cache"], case["block_table"], case["lengths"], case["scale"],
                               k_scale=case["k_scale"], v_scale=case["v_scale"], return_lse=True, **more)


def check_attention(case):
    out, lse = attend(case)
    expected, slack, expected_lse, lse_slack = plain.attention(
        case["q"], case["k_cache"], case["v_cache"], case["k_scale"], case["v_scale"], case["block_table"], case["lengths"], case["scale"])
    plain.close(out, expected, slack)
    plain.close(lse, expected_lse, lse_slack)
    page, table = case["k_cache"].shape[2], case["block_table"]
    if int(case["lengths"].max()) <= table.shape[1] * page:
        # with room for long sequences behind it, which nothing reads, a table's work is split another way
        room = torch.full((table.shape[0], 4096 // page + 1), 2 ** 30, dtype=torch.int32, device=DEV)
        other, other_lse = attend(case | {"block_table": torch.cat([table, room], 1)})
        plain.close(other, expected, slack)
        plain.close(other_lse, expected_lse, lse_slack)
    return out, lse


ATTEND = [  # lengths, kv_heads, group, page, layout
    ([1], 1, 1, 16, "heads"), ([0], 2, 4, 16, "heads"), ([0, 5, 0, 1, 64, 65, 63, 128, 127, 129], 2, 4, 16, "tokens"),
    ([700, 1, 333], 3, 1, 7, "apart"), ([1000, 999], 1, 8, 1, "heads"), ([257, 31, 480], 2, 5, 100, "tokens"),
    ([300, 0, 2], 2, 9, 16, "heads"), ([513, 100], 1, 16, 32, "apart"), ([200, 77], 2, 17, 64, "heads"), ([150], 1, 40, 16, "tokens"),
    ([5000], 1, 4, 64, "heads"), ([20000, 3, 12000], 2, 8, 256, "tokens"), ([2600], 8, 4, 2600, "apart")]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("store", [None, I8, E4M3])
@pytest.mark.parametrize("columns", [64, 128])
@pytest.mark.parametrize("lengths, kv_heads, group, page, layout", ATTEND)
def test_paged_attention(lengths, kv_heads, group, page, layout, columns, store, dtype):
    check_attention(attention_case(lengths, kv_heads, group, columns, page, dtype, store or dtype, layout, seed=len(lengths) + group))
    no_status()


@pytest.mark.parametrize("store", [F16, I8])
@pytest.mark.parametrize("columns", [64, 128])
@pytest.mark.parametrize("batch", [2, 70])
def test_paged_attention_where_tables_begin_to_be_cut(batch, columns, store):
    """Tables of as many positions as a block takes by itself, and of one page more, with few and many sequences."""
    for room in (256, 512):
        for positions in (room, room + 16):
            lengths = [positions, 1] + [(i * 131) % positions for i in range(batch - 2)]
            case = attention_case(lengths, 4, 3, columns, 16, F16, store, "tokens", seed=batch + positions, slack_columns=0)
            check_attention(case)
            results = [attend(case) for _ in range(3)]
            assert all(torch.equal(results[0][0], out) and torch.equal(results[0][1], lse) for out, lse in results)
    no_status()


@pytest.mark.parametrize("batch", [129, 300])
def test_paged_attention_of_many_sequences(batch):
    """More sequences than a block has threads: the scans take several rounds."""
    lengths = [(i * 37) % 90 * (i % 3 != 1) for i in range(batch)]
    for kv_heads, group, store in ((1, 2, F16), (4, 12, E4M3)):
        check_attention(attention_case(lengths, kv_heads, group, 64, 8, F16, store, "tokens", seed=batch))
    no_status()


@pytest.mark.parametrize("store", [BF16, I8, E4M3])
def test_paged_attention_with_a_sharp_softmax_and_uneven_rows(store):
    """Scores of hundreds, a value row 1e4 times the others that nearly nothing attends to, and a row of
    zeros that nearly everything attends to."""
    case = attention_case([900, 64, 333], 2, 4, 128, 16, BF16, store, "heads", seed=4, spread=25.0)
    check_attention(case)
    case = attention_case([400], 1, 4, 128, 16, BF16, store, "heads", seed=5, spread=4.0)
    q = case["q"].float().mean((0, 1))
    for row, key, value in ((3, -2.0, 1e4), (77, 3.0, 0.0), (200, 0.5, 1e-4)):
        slot = int(case["block_table"][0, row // 16]) * 16 + row % 16
        ops.cache_write((key * q).to(BF16).view(1, 1, 128), (value * randn(1, 1, 128, seed=row)).to(BF16),
                        torch.tensor([slot], device=DEV), case["k_cache"], case["v_cache"], case["k_scale"], case["v_scale"])
    check_attention(case)


def test_paged_attention_infinities_and_nan():
    for store in (F16, I8):
        case = attention_case([70, 40], 1, 4, 64, 16, F16, store, "heads", seed=6)
        slot = int(case["block_table"][0, 1]) * 16 + 3
        row = randn(1, 1, 64, dtype=F16, seed=1)
        bad = row.clone()
        bad[..., 9] = float("nan")
        ops.cache_write(bad, row, torch.tensor([slot], device=DEV), case["k_cache"], case["v_cache"], case["k_scale"], case["v_scale"])
        out, lse = attend(case)
        assert out[0].isnan().all() and lse[0].isnan().all() and out[1].isfinite().all()      # the key is NaN
        ops.cache_write(row, bad, torch.tensor([slot], device=DEV), case["k_cache"], case["v_cache"], case["k_scale"], case["v_scale"])
        out, lse = attend(case)
        spoilt = out[0].isnan()
        assert (spoilt.all() if store == I8 else spoilt[:, 9].all() and spoilt.sum() == 4) and lse.isfinite().all()
    # scores of -infinity beside finite ones weigh nothing
    case = attention_case([70], 1, 4, 64, 16, F16, F16, "heads", seed=7)
    case["q"][...] = case["q"].abs() + 0.1
    slot = int(case["block_table"][0, 2]) * 16 + 5
    ops.cache_write(torch.full((1, 1, 64), -float("inf"), dtype=F16, device=DEV), randn(1, 1, 64, dtype=F16),
                    torch.tensor([slot], device=DEV), case["k_cache"], case["v_cache"])
    check_attention(case)


def test_bad_pages_and_lengths_are_left_out_and_reported():
    case = attention_case([200, 64, 90], 2, 4, 64, 16, BF16, BF16, "tokens", seed=8)
    for bad in (-1, case["k_cache"].shape[0], 2 ** 31 - 1, -2 ** 31):
        case["block_table"][1, 2] = bad
        check_attention(case)
        status_names(1)
    case["block_table"][2, :6] = -1                      # nothing of a sequence is there: no sum at all
    out, lse = attend(case)
    with pytest.raises(ValueError):
        ops.workspace_status(DEV)
    assert out[2].isnan().all() and (lse[2] == -float("inf")).all() and out[0].isfinite().all()
    room = torch.full((3, 300), -1, dtype=torch.int32, device=DEV)
    out, lse = attend(case | {"block_table": torch.cat([case["block_table"], room], 1)})
    with pytest.raises(ValueError):
        ops.workspace_status(DEV)
    assert out[2].isnan().all() and (lse[2] == -float("inf")).all() and out[0].isfinite().all()
    case = attention_case([200, 64, 90], 2, 4, 64, 16, BF16, I8, "tokens", seed=9, slack_columns=0)
    for length in (209, 2 ** 31 - 1):
        case["lengths"][0] = length                      # more than the table names: cut to its 208 positions
        case["k_scale"].nan_to_num_(0.01), case["v_scale"].nan_to_num_(0.01)
        check_attention(case)
        status_names(0)
    case["lengths"][0] = -5
    out, lse = check_attention(case)
    no_status()
    assert not out[0].any()
    # no columns at all
    out, lse = ops.paged_attention(case["q"], case["k_cache"], case["v_cache"], case["block_table"][:, :0], int32([0, 0, 0]),
                                   0.1, k_scale=case["k_scale"], v_scale=case["v_scale"], return_lse=True)
    assert not out.any() and (lse == -float("inf")).all()
    no_status()


def test_paged_attention_strides_outputs_and_shared_pages():
    case = attention_case([130, 130, 130], 2, 4, 128, 16, F16, F16, "heads", seed=10)
    case["block_table"][1], case["block_table"][2, :5] = case["block_table"][0], case["block_table"][0, :5].clone()   # shared prefixes
    expected, _ = check_attention(case)
    wide = torch.zeros(3, 20, 256, dtype=F16, device=DEV)
    view = wide[:, 2:18:2, 128:]
    view.copy_(case["q"])
    table = torch.full((3, 2 * case["block_table"].shape[1]), 99999, dtype=torch.int32, device=DEV)[:, ::2]
    table.copy_(case["block_table"])
    lengths = int32([130, 9, 130, 9, 130, 9])[::2]
    target = torch.zeros(8, 3, 192, dtype=F16, device=DEV)
    out = ops.paged_attention(view, case["k_cache"], case["v_cache"], table, lengths, case["scale"], out=target[..., 64:].transpose(0, 1))
    assert torch.equal(out, expected) and not target[..., :64].any()
    assert torch.equal(ops.paged_attention(case["q"], case["k_cache"], case["v_cache"], case["block_table"], case["lengths"],
                                           case["scale"]), expected)
    # one table and one length for all sequences, one query for all heads; a negative scale
    check_attention(case | {"block_table": case["block_table"][:1].expand(3, -1), "lengths": int32([77]).expand(3),
                            "q": case["q"][:, :1].expand(3, 8, 128), "scale": -0.2})
    with pytest.raises(ValueError):
        ops.paged_attention(case["q"], case["k_cache"], case["v_cache"], case["block_table"], case["lengths"], 0.1, out=case["q"])
    with pytest.raises(TypeError):
        ops.paged_attention(case["q"], case["k_cache"], case["v_cache"], case["block_table"].long(), case["lengths"], 0.1)
    with pytest.raises(TypeError):
        ops.paged_attention(case["q"].to(BF16), case["k_cache"], case["v_cache"], case["block_table"], case["lengths"], 0.1)


def test_offsets_past_32_bits():
    """Pages more than 2^32 elements apart."""
    pages, page, columns = 3, 16, 64
    stride = (1 << 31) + 1024
    memory = torch.zeros(2 * stride + 4 * page * columns, dtype=I8, device=DEV)
    kc = memory.as_strided((pages, 2, page, columns), (stride, page * columns, columns, 1))
    vc = memory.as_strided((pages, 2, page, columns), (stride, page * columns, columns, 1), 2 * page * columns)
    scales = torch.full((2, pages, 2, page), float("nan"), device=DEV)
    k, v = cache_rows(40, 2, columns, BF16)
    slots = torch.cat((torch.arange(32, 48), torch.arange(16, 32), torch.arange(0, 8))).to(DEV)
    ops.cache_write(k, v, slots, kc, vc, scales[0], scales[1])
    back = ops.cache_read(kc, vc, slots, scales[0], scales[1], dtype=BF16)
    assert torch.equal(back[0], plain.quantise(k, I8)[0].to(BF16)) and torch.equal(back[1], plain.quantise(v, I8)[0].to(BF16))
    check_attention({"q": randn(1, 8, columns, dtype=BF16), "k_cache": kc, "v_cache": vc, "block_table": int32([[2, 1, 0]]),
                     "lengths": int32([40]), "scale": 0.125, "k_scale": scales[0], "v_scale": scales[1]})
    no_status()


def test_results_do_not_vary_and_calls_overlap_on_streams():
    cases = [attention_case([3000, 17, 900], 2, 4, 128, 16, BF16, store, "heads", seed=11 + i)
             for i, store in enumerate((BF16, I8, E4M3, BF16))]
    expected = [attend(case) for case in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    got = [[] for _ in cases]
    for _ in range(20):
        for stream, case, results in zip(streams, cases, got):
            with torch.cuda.stream(stream):
                results.append(attend(case))
    torch.cuda.synchronize()
    for want, results in zip(expected, got):
        assert all(torch.equal(want[0], out) and torch.equal(want[1], lse) for out, lse in results)


def test_in_a_graph_with_new_contents():
    """Captured calls follow what their buffers hold at each replay; two graphs share nothing."""
    ops.workspace(DEV)
    first = attention_case([600, 5, 0, 2000], 2, 4, 128, 16, BF16, E4M3, "heads", seed=21)
    second = attention_case([100, 1500, 30, 2000], 2, 4, 128, 16, BF16, E4M3, "heads", seed=22)
    graphs, results = [], []
    for case in (first, second):
        attend(case)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(attend(case))
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for case, (out, lse) in zip((first, second), results):
        want = attend(case)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    first["lengths"].copy_(int32([1, 5, 0, 1999]))
    first["q"].mul_(0.5)
    graphs[0].replay()
    want = attend(first)
    torch.cuda.synchronize()
    assert torch.equal(results[0][0], want[0]) and torch.equal(results[0][1], want[1])
    q, k, qw, kw, cos, sin, positions = rotary_inputs(33, 8, 2, 64, 32, F32)
    gq, gk = randn(33, 8, 64), randn(33, 2, 64)
    ops.head_norm_rotary_backward(gq, gk, q, k, qw, kw, cos, sin, positions)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.head_norm_rotary_backward(gq, gk, q, k, qw, kw, cos, sin, positions)
    gq.mul_(2)
    positions[4] = -1
    graph.replay()
    want = ops.head_norm_rotary_backward(gq, gk, q, k, qw, kw, cos, sin, positions)
    assert all(torch.equal(a, b) for a, b in zip(held, want))
    no_status()


def test_in_a_graph_behind_copies_and_other_streams():
    """Kernels that may be placed early keep the order that the stream gives them: behind a copy, behind a fill,
    behind two streams at once, eagerly and captured."""
    case = attention_case([300, 77], 2, 4, 128, 16, BF16, I8, "heads", seed=31)
    q, k, qw, kw, cos, sin, positions = rotary_inputs(2, 8, 2, 128, 64, BF16, seed=32)
    next_q, next_k = [randn(*t.shape, dtype=BF16, seed=40 + i) for i, t in enumerate((q, k))]
    v = randn(2, 2, 128, dtype=BF16, seed=33)
    slots = torch.zeros(2, dtype=torch.int64, device=DEV)
    for b, n in enumerate((300, 77)):
        slots[b] = int(case["block_table"][b, n // 16]) * 16 + n % 16 if n % 16 else -1
    case["lengths"] = int32([300 + (300 % 16 > 0), 77 + (77 % 16 > 0)])
    held = [t.clone() for t in (case["k_cache"], case["v_cache"], case["k_scale"], case["v_scale"])]
    staged_q, staged_k, staged_v = torch.empty_like(next_q), torch.empty_like(next_k), torch.empty_like(v)

    def work(side):
        main = torch.cuda.current_stream()
        staged_q.copy_(next_q)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            staged_v.fill_(0)
            staged_v.copy_(v)
        staged_k.copy_(next_k)
        turned = ops.head_norm_rotary(staged_q, staged_k, qw, kw, cos, sin, positions)
        main.wait_stream(side)
        ops.cache_write(turned[1], staged_v, slots, case["k_cache"], case["v_cache"], case["k_scale"], case["v_scale"])
        out, lse = attend(case | {"q": turned[0]})
        grads = ops.head_norm_rotary_backward(turned[0], turned[1], staged_q, staged_k, qw, kw, cos, sin, positions)
        back = ops.cache_read(case["k_cache"], case["v_cache"], slots, case["k_scale"], case["v_scale"], dtype=BF16)
        staged_q.fill_(float("nan"))          # behind all readers
        staged_k.fill_(float("nan"))
        return (*turned, out, lse, *grads, *back)

    want = [t.clone() for t in work(torch.cuda.Stream())]
    torch.cuda.synchronize()
    assert all(t.isfinite().all() for t in want)
    plain.close(want[0], *plain.norm_rotary(next_q, qw, cos, sin, positions, 1e-6, False))
    for t, old in zip((case["k_cache"], case["v_cache"], case["k_scale"], case["v_scale"]), held):
        t.copy_(old)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.graph(graph):
        got = work(side)
    for _ in range(20):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):                       # eagerly, back to back, on streams in turn
        for stream in streams:
            stream.wait_stream(streams[0] if stream is streams[1] else streams[1])
            with torch.cuda.stream(stream):
                again = work(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    no_status()


# -------------------------------------------------------------------------- all of them in a row
@pytest.mark.parametrize("store", [BF16, I8, E4M3])
def test_a_prompt_and_new_tokens(store):
    """A prompt of two sequences and four steps: norm and rotation, the cache, attention; the prompt through
    ops.flash_attention.  Each step's output against the plain forms over the same rounded rows."""
    heads, kv_heads, columns, page, prompt = 8, 2, 128, 16, 128
    qw, kw = (1 + 0.2 * randn(2, columns, seed=1)).to(BF16)
    angle = torch.arange(512, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, columns, 2, device=DEV).double() / columns)
    cos, sin = angle.cos().float(), angle.sin().float()
    kc, vc, ks, vs = plain.new_cache(40, kv_heads, page, columns, store, "tokens", DEV)
    table = torch.randperm(40, generator=torch.Generator().manual_seed(2))[:32].reshape(2, 16).to(DEV, torch.int32)
    scale = columns ** -0.5
    keys, vals = [], []
    for step in range(5):
        new = prompt if step == 0 else 1
        past = 0 if step == 0 else prompt + step - 1
        qkv = randn(2 * new, heads + 2 * kv_heads, columns, dtype=BF16, seed=50 + step)
        q, k, v = qkv.split((heads, kv_heads, kv_heads), 1)
        positions = (past + torch.arange(new, device=DEV)).repeat(2).to(torch.int32)
        turned_q, turned_k = ops.head_norm_rotary(q, k, qw, kw, cos, sin, positions)
        plain.close(turned_q, *plain.norm_rotary(q, qw, cos, sin, positions, 1e-6, False))
        plain.close(turned_k, *plain.norm_rotary(k, kw, cos, sin, positions, 1e-6, False))
        slots = torch.cat([table[b].long()[positions[:new].long() // page] * page + positions[:new] % page for b in range(2)])
        ops.cache_write(turned_k, v, slots, kc, vc, ks, vs)
        keys.append(turned_k.reshape(2, new, kv_heads, columns))
        vals.append(v.reshape(2, new, kv_heads, columns))
        if step == 0:
            whole = [t.reshape(2, new, -1, columns).transpose(1, 2).contiguous() for t in (turned_q, turned_k, v)]
            prompt_out = ops.flash_attention(*whole, scale, head_group=heads // kv_heads)
            last_q = whole[0][:, :, -1].contiguous()
        else:
            last_q = turned_q
        lengths = int32([past + new] * 2)
        out, lse = ops.paged_attention(last_q, kc, vc, table, lengths, scale, k_scale=ks, v_scale=vs, return_lse=True)
        expected, slack, expected_lse, lse_slack = plain.attention(last_q, kc, vc, ks, vs, table, lengths, scale)
        plain.close(out, expected, slack)
        plain.close(lse, expected_lse, lse_slack)
        # and against the rows that went in: exactly in 16 bits, within the codes' steps in 8
        held_k, held_v = torch.cat(keys, 1), torch.cat(vals, 1)
        query = last_q.double().reshape(2, kv_heads, heads // kv_heads, columns)
        weights = torch.softmax(torch.einsum("bhgd,blhd->bhgl", query, held_k.double()) * scale, -1)
        unrounded = torch.einsum("bhgl,blhd->bhgd", weights, held_v.double()).reshape(2, heads, columns)
        error = (out.double() - unrounded).norm() / unrounded.norm()
        assert error <= {BF16: 2.0 ** -8, I8: 2.0 ** -5, E4M3: 2.0 ** -3}[store]
        if step == 0 and store == BF16:
            assert (out.double() - prompt_out[:, :, -1].double()).norm() <= 1e-2 * out.double().norm()
        rows = torch.cat([table[b].long()[:, None] * page + torch.arange(page, device=DEV) for b in range(2)]).reshape(2, -1)[:, :past + new]
        back_k, back_v = ops.cache_read(kc, vc, rows.reshape(-1), ks, vs, dtype=BF16)
        for back, held in ((back_k, held_k), (back_v, held_v)):
            exact = held.double() if store == BF16 else plain.quantise(held, store)[0]
            assert torch.equal(back.reshape(held.shape), exact.float().to(BF16))
    no_status()
