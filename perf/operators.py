"""What is measured of the operators around a key-value cache: per-head norm and rotation (forward
and backward), writing and reading a paged cache in 16 and 8 bits, and attention of one new token
over that cache.  ``run`` computes them in elementary torch operations, or, with ``own``, through
``intent_b200.ops``; ``exact`` computes the same values in 64 bits.
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
         "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
WIDTH = {"f32": 4, "f16": 2, "bf16": 2, "int8": 1, "e4m3": 1}
TINY = 2.0 ** -126


# ------------------------------------------------------------------------------------- cases
def _rotary(name, op, tokens, heads, kv_heads, dim, rotated, dtype, interleaved=False, padded=0, past=0):
    return {"name": name, "op": op, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotated": rotated, "dtype": dtype, "interleaved": interleaved, "padded": padded, "past": past}


def _cache(name, op, tokens, kv_heads, dim, dtype, store, page, pages, token_major, padded=0):
    return {"name": name, "op": op, "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "store": store, "page": page, "pages": pages, "token_major": token_major, "padded": padded}


def _attend(name, batch, kv_heads, group, dim, longest, shortest, dtype, store, page, token_major, empty=0):
    return {"name": name, "op": "attend", "batch": batch, "kv_heads": kv_heads, "group": group, "dim": dim,
            "longest": longest, "shortest": shortest, "dtype": dtype, "store": store, "page": page,
            "token_major": token_major, "empty": empty}


def listed():
    return [
        # one decoding step of eight sequences far into their text: the latency of the call counts
        _rotary("rotary step of 8", "rotary", 8, 32, 8, 128, 128, "bf16", past=100000),
        # the prompt of eight sequences of 2048 tokens
        _rotary("rotary prompt 16384", "rotary", 16384, 32, 8, 128, 128, "bf16"),
        # the training step on the same batch
        _rotary("rotary backward 16384", "rotary_backward", 16384, 32, 8, 128, 128, "bf16"),
        # a small ragged training batch in f32 whose heads rotate half of their dimensions, with padding behind it
        _rotary("rotary backward ragged", "rotary_backward", 1001, 12, 4, 64, 32, "f32", interleaved=True, padded=23),
        # a prompt of eight sequences of 4096 tokens goes into a 16-bit cache
        _cache("cache write 32768", "write", 32768, 8, 128, "bf16", "bf16", 16, 2100, True),
        # the same prompt is quantised into an 8-bit cache and the cache read back for the prompt's next piece
        _cache("cache int8 32768", "write_read", 32768, 8, 128, "bf16", "int8", 64, 516, False),
        # a short odd chunk, padded to its batch's shape, in the other 8-bit type
        _cache("cache e4m3 chunk", "write_read", 77, 2, 64, "f16", "e4m3", 16, 8, True, padded=5),
        # one long text: few rows, so the cache's length is what there is to split
        _attend("attend one of 131072", 1, 8, 4, 128, 131072, 131072, "bf16", "bf16", 64, False),
        # a serving batch of ragged lengths
        _attend("attend 64 ragged", 64, 8, 4, 128, 4096, 100, "bf16", "bf16", 16, True),
        # the same with an 8-bit cache and longer texts
        _attend("attend 64 e4m3", 64, 8, 4, 128, 8192, 1000, "bf16", "e4m3", 16, True),
        # many query heads on two key heads, 8-bit whole numbers
        _attend("attend 16 int8 grouped", 16, 2, 16, 128, 4096, 1, "f16", "int8", 32, False),
        # short texts, a key head for each query head, some sequences not begun
        _attend("attend 8 short", 8, 32, 1, 64, 300, 1, "f16", "f16", 16, False, empty=2),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case of the same ranges, at most as costly as the largest listed one of its kind."""
    op = rng.choice(["rotary", "rotary_backward", "write", "write_read", "attend", "attend"])
    if op.startswith("rotary"):
        dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
        rotated = rng.choice([dim, dim, 16 * rng.randint(1, dim // 16)])
        kv_heads, group = rng.randint(1, 8), rng.choice([1, 2, 3, 4, 8])
        dtype = rng.choice(["bf16", "f16", "f32"])
        most = 16384 * 40 * 128 * 2 // (kv_heads * (group + 1) * dim * WIDTH[dtype])
        tokens = _log(rng, 1, min(most, 16384))
        padded = rng.choice([0, rng.randint(0, tokens // 4)])
        return _rotary("", op, tokens, kv_heads * group, kv_heads, dim, rotated, dtype,
                       rng.random() < 0.4, padded, rng.choice([0, _log(rng, 1, 130000)]))
    dim = rng.choice([64, 128])
    page = rng.choice([1, 8, 16, 16, 32, 64, 100])
    dtype = rng.choice(["bf16", "f16"])
    store = rng.choice([dtype, "int8", "e4m3"])
    token_major = rng.random() < 0.5
    if op.startswith("write"):
        kv_heads = rng.randint(1, 16)
        tokens = _log(rng, 1, 32768 * 8 * 128 // (kv_heads * dim))
        store = dtype if op == "write" else rng.choice(["int8", "e4m3"])
        pages = -(-tokens // page) + rng.randint(0, 4)
        return _cache("", op, tokens, kv_heads, dim, dtype, store, page, pages, token_major,
                      rng.choice([0, rng.randint(0, tokens // 4)]))
    batch, kv_heads = _log(rng, 1, 128), rng.randint(1, 16)
    group = rng.choice([1, 2, 4, 5, 8, 12, 16, 24])
    most = min(131072, 64 * 4096 * 8 * 128 // (batch * kv_heads * dim), 64 * 4096 * 8 * 4 // (batch * kv_heads * group))
    longest = _log(rng, 1, max(1, most))
    shortest = rng.choice([longest, rng.randint(1, longest)])
    return _attend("", batch, kv_heads, group, dim, longest, shortest, dtype, store, page, token_major,
                   rng.choice([0, rng.randint(0, batch // 2)]))


# ------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _randn(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype)


def _tables(rows, rotated):
    """cos and sin of position * 10000^(-2i/rotated), angles in 64 bits."""
    rate = 10000.0 ** (-torch.arange(0, rotated, 2, device=DEVICE, dtype=torch.float64) / rotated)
    angle = torch.arange(rows, device=DEVICE, dtype=torch.float64)[:, None] * rate[None, :]
    return torch.cos(angle).float(), torch.sin(angle).float()


def _prepare_rotary(c, g):
    dtype, tokens = TYPES[c["dtype"]], c["tokens"]
    # q and k are the leading columns of one projection's output, as a fused projection gives them
    both = _randn((tokens, c["heads"] + 2 * c["kv_heads"], c["dim"]), g, dtype)
    q, k = both[:, :c["heads"]], both[:, c["heads"]:c["heads"] + c["kv_heads"]]
    state = {"case": c, "q": q, "k": k, "epsilon": 1e-6,
             "q_weight": (1 + 0.2 * _randn((c["dim"],), g)).to(dtype), "k_weight": (1 + 0.2 * _randn((c["dim"],), g)).to(dtype)}
    length = min(2048, max(1, tokens))
    state["cos"], state["sin"] = _tables(c["past"] + length, c["rotated"])
    positions = c["past"] + torch.arange(tokens, device=DEVICE, dtype=torch.int64) % length
    if c["op"] == "rotary" and tokens <= 128:   # a step: every sequence is at a place of its own
        positions = torch.randint(0, c["past"] + length, (tokens,), generator=g, device=DEVICE)
    if c["padded"]:
        positions[tokens - c["padded"]:] = -1
    state["positions"] = positions.to(torch.int32)
    if c["op"] == "rotary_backward":
        state["grad_q"] = _randn((tokens, c["heads"], c["dim"]), g, dtype)
        state["grad_k"] = _randn((tokens, c["kv_heads"], c["dim"]), g, dtype)
    return state


def _empty_cache(pages, kv_heads, page, dim, store, token_major):
    """A cache whose unwritten slots hold what memory may hold: NaN, and codes under a NaN scale."""
    order = (pages, page, kv_heads, dim) if token_major else (pages, kv_heads, page, dim)
    cache = torch.full(order, float("nan"), device=DEVICE, dtype=TYPES[store]) if WIDTH[store] == 2 else \
        torch.full(order, 85, device=DEVICE, dtype=torch.int8).view(TYPES[store])
    scale = None if WIDTH[store] == 2 else torch.full(order[:3], float("nan"), device=DEVICE)
    if token_major:
        cache, scale = cache.transpose(1, 2), None if scale is None else scale.transpose(1, 2)
    return cache, scale


def _prepare_cache(c, g):
    tokens, capacity, dtype = c["tokens"], c["page"] * c["pages"], TYPES[c["dtype"]]
    # a projection's output again: rows further apart than they are long, each key head of a size of its own
    size = torch.exp(_randn((1, 2 * c["kv_heads"], 1), g)) * torch.exp(0.3 * _randn((tokens, 2 * c["kv_heads"], 1), g))
    both = (size * _randn((tokens, 2 * c["kv_heads"], c["dim"]), g)).to(dtype)
    slots = torch.randperm(c["pages"], generator=g, device=DEVICE)[:, None] * c["page"] + \
        torch.arange(c["page"], device=DEVICE)[None, :]
    slots = slots.reshape(-1)[:tokens].clone()   # pages in any order, filled one after the other
    if c["padded"]:
        slots[tokens - c["padded"]:] = -1
    state = {"case": c, "k": both[:, :c["kv_heads"]], "v": both[:, c["kv_heads"]:], "slots": slots}
    state["k_cache"], state["k_scale"] = _empty_cache(c["pages"], c["kv_heads"], c["page"], c["dim"], c["store"], c["token_major"])
    state["v_cache"], state["v_scale"] = _empty_cache(c["pages"], c["kv_heads"], c["page"], c["dim"], c["store"], c["token_major"])
    if c["op"] == "write_read":
        for name in ("k_scale", "v_scale"):   # an older text's rows fill the other slots
            state[name].fill_(1.0 / 64)
        state["all"] = torch.arange(capacity, device=DEVICE)
    return state


def _lengths(c, g):
    span = c["longest"] - c["shortest"] + 1
    lengths = c["shortest"] + (torch.rand((c["batch"],), generator=g, device=DEVICE) * span).long().clamp_(max=span - 1)
    lengths[0] = c["longest"]
    if c["empty"]:
        lengths[c["batch"] - c["empty"]:] = 0
    return lengths


def _prepare_attend(c, g):
    dtype, page = TYPES[c["dtype"]], c["page"]
    lengths = _lengths(c, g)
    columns = -(-c["longest"] // page)
    held = (lengths + page - 1) // page
    pages = c["batch"] * columns
    # every sequence's pages lie anywhere in the cache; the table's columns behind a sequence hold -1
    table = torch.randperm(pages, generator=g, device=DEVICE).reshape(c["batch"], columns)
    column = torch.arange(columns, device=DEVICE)
    state = {"case": c, "lengths": lengths.to(torch.int32), "scale": c["dim"] ** -0.5,
             "block_table": torch.where(column[None, :] < held[:, None], table, -1).to(torch.int32)}
    state["q"] = (1.5 * _randn((c["batch"], c["kv_heads"] * c["group"], c["dim"]), g)).to(dtype)
    inside = (column[None, :, None] * page + torch.arange(page, device=DEVICE) < lengths[:, None, None])
    written = torch.empty((pages, page), dtype=torch.bool, device=DEVICE)
    written[table.reshape(-1)] = inside.reshape(pages, page)
    for name in ("k", "v"):
        cache, scale = _empty_cache(pages, c["kv_heads"], page, c["dim"], c["store"], c["token_major"])
        size = torch.exp(0.3 * _randn((pages, c["kv_heads"], page), g))
        here = written[:, None, :]
        if scale is None:
            for at in range(0, pages, 1 + (1 << 26) // (c["kv_heads"] * page * c["dim"])):
                to = slice(at, at + 1 + (1 << 26) // (c["kv_heads"] * page * c["dim"]))
                rows = size[to, ..., None] * _randn((*size[to].shape, c["dim"]), g)
                cache[to] = torch.where(here[to, ..., None], rows, float("nan")).to(cache.dtype)
        else:
            for at in range(0, pages, 1 + (1 << 26) // (c["kv_heads"] * page * c["dim"])):
                to = slice(at, at + 1 + (1 << 26) // (c["kv_heads"] * page * c["dim"]))
                rows = _randn((*size[to].shape, c["dim"]), g)
                # codes as a row's quantisation leaves them, their largest near the type's end
                if c["store"] == "int8":
                    cache[to] = (rows * 36).round().clamp(-127, 127).to(torch.int8)
                else:
                    cache.view(torch.int8)[to] = (rows * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.int8)
            scale.copy_(torch.where(here, size * (1 / 36 if c["store"] == "int8" else 2.0 ** -7), float("nan")))
        state[name + "_cache"], state[name + "_scale"] = cache, scale
    return state


def prepare(case, seed):
    g = _generator(seed)
    if case["op"].startswith("rotary"):
        return _prepare_rotary(case, g)
    if case["op"] == "attend":
        return _prepare_attend(case, g)
    return _prepare_cache(case, g)


# ------------------------------------------------------------------------------- plain forms
def _rotate(x, cos, sin, interleaved, back):
    """R x (R^T x with `back`) on the first 2 * cos.shape[-1] columns of x (tokens, heads, dim)."""
    half = cos.shape[-1]
    cos, sin = cos[:, None], (-sin if back else sin)[:, None]
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _norm_rotary(x, weight, cos, sin, live, epsilon, interleaved):
    wide = x.float()
    rstd = torch.rsqrt((wide * wide).mean(-1, keepdim=True) + epsilon)
    y = _rotate(wide * rstd * weight.float(), cos, sin, interleaved, False)
    return torch.where(live, y, 0.0).to(x.dtype)


def _norm_rotary_backward(grad, x, weight, cos, sin, live, epsilon, interleaved):
    wide = x.float()
    rstd = torch.rsqrt((wide * wide).mean(-1, keepdim=True) + epsilon)
    xhat = wide * rstd
    g = torch.where(live, _rotate(grad.float(), cos, sin, interleaved, True), 0.0)
    u = g * weight.float()
    dx = rstd * (u - xhat * (u * xhat).mean(-1, keepdim=True))
    return dx.to(x.dtype), (g * xhat).sum(0).sum(0)


def _run_rotary(s):
    c = s["case"]
    live = (s["positions"] >= 0)[:, None, None]
    at = s["positions"].clamp(min=0).long()
    cos, sin = s["cos"][at], s["sin"][at]
    if c["op"] == "rotary":
        return (_norm_rotary(s["q"], s["q_weight"], cos, sin, live, s["epsilon"], c["interleaved"]),
                _norm_rotary(s["k"], s["k_weight"], cos, sin, live, s["epsilon"], c["interleaved"]))
    dq, dwq = _norm_rotary_backward(s["grad_q"], s["q"], s["q_weight"], cos, sin, live, s["epsilon"], c["interleaved"])
    dk, dwk = _norm_rotary_backward(s["grad_k"], s["k"], s["k_weight"], cos, sin, live, s["epsilon"], c["interleaved"])
    return dq, dk, dwq, dwk


def _quantise(x, store):
    """(codes, scale) of rows; the quotients next to a border need 64 bits."""
    amax = x.double().abs().amax(-1)
    if store == "int8":
        scale = (amax / 127).float().clamp(min=TINY)
        codes = torch.round(x.double() / scale.double()[..., None])
    else:
        mantissa, exponent = torch.frexp(amax)
        exponent = torch.where(amax > 0, exponent - 9 + (mantissa > 0.875), -126).clamp(min=-126)
        scale = torch.ldexp(torch.ones_like(amax), exponent).float()
        codes = x.float() / scale[..., None]
    fine = torch.isfinite(amax)
    codes = torch.where(fine[..., None], codes, 0.0)
    return codes.to(TYPES[store]), torch.where(fine, scale, float("nan"))


def _write(rows, slots, cache, scale, store, page):
    live = slots >= 0
    slots, rows = slots[live], rows[live]
    at = (slots // page, slice(None), slots % page)
    if scale is None:
        cache[at] = rows
    else:
        codes, size = _quantise(rows, store)
        cache.view(torch.int8)[at] = codes.view(torch.int8)
        scale[at] = size


def _read(slots, cache, scale, page, dtype):
    at = (slots // page, slice(None), slots % page)
    return (cache.view(torch.int8)[at].view(cache.dtype).float() * scale[at][..., None]).to(dtype)


def _run_cache(s):
    c = s["case"]
    _write(s["k"], s["slots"], s["k_cache"], s["k_scale"], c["store"], c["page"])
    _write(s["v"], s["slots"], s["v_cache"], s["v_scale"], c["store"], c["page"])
    if c["op"] == "write":
        return s["k_cache"], s["v_cache"]
    # the whole cache, as the values that it stands for
    return (_read(s["all"], s["k_cache"], s["k_scale"], c["page"], s["k"].dtype),
            _read(s["all"], s["v_cache"], s["v_scale"], c["page"], s["v"].dtype))


def _gather(cache, scale, table, live):
    """(batch, kv_heads, columns * page, dim) in f32, zeros where nothing is."""
    small = cache.element_size() == 1
    rows = (cache.view(torch.int8) if small else cache)[table]
    rows = (rows.view(cache.dtype) if small else rows).float()
    if scale is not None:
        rows = rows * scale[table][..., None]
    rows = rows.transpose(1, 2).flatten(2, 3)
    return torch.where(live, rows, 0.0)


def _run_attend(s):
    c = s["case"]
    table = s["block_table"].clamp(min=0).long()
    key = torch.arange(table.shape[1] * c["page"], device=table.device)
    live = key[None, :] < s["lengths"][:, None]
    k = _gather(s["k_cache"], s["k_scale"], table, live[:, None, :, None])
    v = _gather(s["v_cache"], s["v_scale"], table, live[:, None, :, None])
    q = s["q"].float().unflatten(1, (c["kv_heads"], c["group"]))
    scores = (q @ k.transpose(-1, -2)) * s["scale"]
    live = live[:, None, None, :]
    scores = torch.where(live, scores, float("-inf"))
    m = scores.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)
    p = torch.exp(scores - m)
    total = p.sum(-1, keepdim=True)
    begun = (s["lengths"] > 0)[:, None, None, None]
    out = torch.where(begun, (p @ v) / total, 0.0).flatten(1, 2)
    lse = (m + torch.log(total)).flatten(1)
    return out.to(s["q"].dtype), lse


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state)
    if op.startswith("rotary"):
        return _run_rotary(state)
    return _run_attend(state) if op == "attend" else _run_cache(state)


def _own(s):
    from intent_b200 import ops
    c = s["case"]
    if c["op"] == "rotary":
        return ops.head_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["positions"],
                                    s["epsilon"], interleaved=c["interleaved"])
    if c["op"] == "rotary_backward":
        return ops.head_norm_rotary_backward(s["grad_q"], s["grad_k"], s["q"], s["k"], s["q_weight"], s["k_weight"],
                                             s["cos"], s["sin"], s["positions"], s["epsilon"], interleaved=c["interleaved"])
    if c["op"] == "attend":
        return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["lengths"], s["scale"],
                                   k_scale=s["k_scale"], v_scale=s["v_scale"], return_lse=True)
    ops.cache_write(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if c["op"] == "write":
        return s["k_cache"], s["v_cache"]
    return ops.cache_read(s["k_cache"], s["v_cache"], s["all"], s["k_scale"], s["v_scale"], dtype=s["k"].dtype)


# -------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"].startswith("rotary"):
        rows, width = c["tokens"] * (c["heads"] + c["kv_heads"]), WIDTH[c["dtype"]]
        passes = 2 if c["op"] == "rotary" else 3
        tables = min(c["tokens"], c["past"] + 2048) * c["rotated"] * 4
        sums = 2 * c["dim"] * (width + (4 if passes == 3 else 0))
        return {"bytes": passes * rows * c["dim"] * width + tables + 4 * c["tokens"] + sums,
                "flops": (8 if passes == 2 else 16) * rows * c["dim"]}
    if c["op"] == "attend":
        lengths = (c["shortest"] + c["longest"]) / 2 * (c["batch"] - c["empty"] - 1) + c["longest"]
        row = 2 * (c["dim"] * WIDTH[c["store"]] + (4 if WIDTH[c["store"]] == 1 else 0))
        heads = c["kv_heads"] * c["group"]
        return {"bytes": lengths * (c["kv_heads"] * row + 4 / c["page"]) + c["batch"] * heads * (c["dim"] * 4 + 4),
                "flops": 4 * heads * c["dim"] * lengths}
    rows = 2 * c["kv_heads"]
    live, capacity = c["tokens"] - c["padded"], c["page"] * c["pages"]
    width, scale = WIDTH[c["store"]], 0 if WIDTH[c["store"]] == 2 else 4
    moved = live * rows * (c["dim"] * (2 + width) + scale) + 8 * c["tokens"]
    if c["op"] == "write_read":
        moved += capacity * rows * (c["dim"] * (2 + width) + scale) + 8 * capacity
    return {"bytes": moved, "flops": 4 * rows * c["dim"] * c["tokens"]}


# ------------------------------------------------------------------------------------- exact
def _exact_rotary(s):
    """Pairs as complex numbers, turned by cos + i sin."""
    c = s["case"]
    half, dim = c["rotated"] // 2, c["dim"]
    i = torch.arange(half, device=DEVICE)
    first, second = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
    live = s["positions"] >= 0
    at = torch.where(live, s["positions"], 0).long()
    unit = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None, :]

    def turn(x, by):
        z = torch.complex(x[..., first], x[..., second]) * by
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    def norm(x):
        return torch.sqrt((x ** 2).sum(-1, keepdim=True) / dim + s["epsilon"])

    outputs, sums = [], []
    for name in ("q", "k"):
        x, w = s[name].double(), s[name + "_weight"].double()
        if c["op"] == "rotary":
            y = turn(x / norm(x) * w, unit)
            y[~live] = 0
            outputs.append(y)
            continue
        g = turn(s["grad_" + name].double(), unit.conj())
        g[~live] = 0
        r = norm(x)
        outputs.append(g * w / r - x * ((g * w * x).sum(-1, keepdim=True) / (dim * r ** 3)))
        sums.append(torch.einsum("thd,thd->d", g, x / r))
    return (*outputs, *sums)


def _exact_rows(x, store):
    """The values that the quantised rows stand for."""
    x = x.double()
    amax = x.abs().max(-1, keepdim=True).values
    if store == "int8":
        scale = torch.clamp((amax / 127).float().double(), min=TINY)
        return torch.round(x / scale) * scale
    scale = torch.exp2(torch.ceil(torch.log2(torch.clamp(amax, min=1e-60) / 448)).clamp(min=-126))
    scale = torch.where(amax > 448 * scale, 2 * scale, torch.where(amax <= 224 * scale, scale / 2, scale)).clamp(min=TINY)
    y = x / scale
    step = torch.exp2(torch.floor(torch.log2(torch.clamp(y.abs(), min=2.0 ** -6))) - 3)   # three bits behind the first
    return torch.round(y / step) * step * scale


def _exact_cache(s):
    c = s["case"]
    found = []
    for name in ("k", "v"):
        cache = s[name + "_cache"]
        wide = cache.double() if cache.element_size() == 2 else cache.float().double() * s[name + "_scale"].double()[..., None]
        wide = wide.clone()
        live = (s["slots"] >= 0).nonzero().flatten()
        page, place = s["slots"][live] // c["page"], s["slots"][live] % c["page"]
        rows = s[name][live].double() if c["op"] == "write" else _exact_rows(s[name][live], c["store"])
        wide[page, :, place] = rows
        # whole: the cache itself, or all slots in their order
        found.append(wide if c["op"] == "write" else wide.permute(0, 2, 1, 3).reshape(-1, c["kv_heads"], c["dim"]))
    return tuple(found)


def _exact_attend(s):
    c = s["case"]
    heads = c["kv_heads"] * c["group"]
    out = torch.zeros((c["batch"], heads, c["dim"]), dtype=torch.float64, device=DEVICE)
    lse = torch.full((c["batch"], heads), float("-inf"), dtype=torch.float64, device=DEVICE)
    lengths = s["lengths"].tolist()
    for b, length in enumerate(lengths):
        if not length:
            continue
        pages = s["block_table"][b, :-(-length // c["page"])].long()
        rows = []
        for name in ("k", "v"):
            cache = s[name + "_cache"]
            part = cache.view(torch.int8)[pages].view(cache.dtype).float() if cache.element_size() == 1 else cache[pages]
            part = part.double()
            if s[name + "_scale"] is not None:
                part = part * s[name + "_scale"][pages].double()[..., None]
            rows.append(part.permute(1, 0, 2, 3).reshape(c["kv_heads"], -1, c["dim"])[:, :length])
        scores = torch.einsum("hgd,hld->hgl", s["q"][b].double().reshape(c["kv_heads"], c["group"], c["dim"]), rows[0]) * s["scale"]
        lse[b] = torch.logsumexp(scores, -1).reshape(-1)
        out[b] = torch.einsum("hgl,hld->hgd", torch.softmax(scores, -1), rows[1]).reshape(heads, c["dim"])
    return out, lse


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"].startswith("rotary"):
        return _exact_rotary(state)
    return _exact_attend(state) if case["op"] == "attend" else _exact_cache(state)
