"""Plain 64-bit forms of the operators around a key-value cache, and how far a kernel may be from them.

A kernel works in f32 and rounds once, so a result may be off by half a step of its type, and by the
f32 errors of what it was computed from; the bounds below count those, from the inputs alone.
"""
import torch

F32 = 2.0 ** -24     # half a step of f32, relative
CODES = (torch.int8, torch.float8_e4m3fn)


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def close(actual, expected, slack) -> None:
    """|a - e| <= half a step of a's type + slack (a tensor or number), element by element; NaN and
    infinities in the same places."""
    a, e = actual.double(), expected.to(actual.device)
    slack = torch.as_tensor(slack, dtype=torch.float64, device=a.device)
    tiny = torch.finfo(actual.dtype).smallest_normal * torch.finfo(actual.dtype).eps    # a subnormal's step
    assert a.shape == e.shape
    assert torch.equal(a.isnan(), e.isnan()), "NaN in other places"
    assert torch.equal(a.isinf(), e.isinf()) and torch.equal(a[a.isinf()], e[e.isinf()]), "infinities in other places"
    bound = half_step(actual.dtype) * e.abs() * 1.001 + slack + tiny
    off = ((a - e).abs() > bound) & e.isfinite()
    if off.any():
        at = tuple(off.nonzero()[0].tolist())
        raise AssertionError(f"{int(off.sum())} of {off.numel()} values are off, first at {at}: {a[at].item()} for "
                             f"{e[at].item()}, allowed {bound.expand_as(e)[at].item()}")


# ------------------------------------------------------------------------- norm and rotation
def rotate(x, cos, sin, interleaved):
    """R x for (tokens, heads, columns) and (tokens, pairs), in x's precision."""
    pairs = cos.shape[-1]
    i = torch.arange(pairs, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
    cos, sin = cos[:, None], sin[:, None]
    y = x.clone()
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    return y


def tables_at(cos, sin, positions):
    live = (positions >= 0) & (positions < cos.shape[0])
    at = torch.where(live, positions, 0).long()
    return live, cos.double()[at], sin.double()[at]


def norm_rotary(x, weight, cos, sin, positions, epsilon, interleaved):
    """(y, slack): y = R(position) (x / rms(x) * weight), zeros for padding."""
    live, c, s = tables_at(cos, sin, positions)
    wide = x.double()
    z = wide / torch.sqrt((wide ** 2).mean(-1, keepdim=True) + epsilon) * weight.double()
    y = rotate(z, c, s, interleaved)
    y = torch.where(live[:, None, None], y, 0.0)
    # mean of squares, root, quotient, two products and the rotation's three roundings: 16 half steps of
    # numbers that are at most the row's largest |z| twice
    return y, 32 * F32 * torch.where(live[:, None, None], z, 0.0).abs().amax(-1, keepdim=True)


def norm_rotary_backward(grad, x, weight, cos, sin, positions, epsilon, interleaved):
    """(dx, its slack, dweight, its slack) from the formulas."""
    live, c, s = tables_at(cos, sin, positions)
    wide = x.double()
    r = 1 / torch.sqrt((wide ** 2).mean(-1, keepdim=True) + epsilon)
    xhat = wide * r
    g = torch.where(live[:, None, None], rotate(grad.double(), c, -s, interleaved), 0.0)
    u = g * weight.double()
    dx = r * (u - xhat * (u * xhat).mean(-1, keepdim=True))
    size = r * (2 * u.abs().amax(-1, keepdim=True) + 2 * xhat.abs().amax(-1, keepdim=True) * (u * xhat).abs().mean(-1, keepdim=True))
    terms = (g * xhat).abs().sum((0, 1))
    # dx: the sums of up to 256 products add 16 in a row, then in a tree: 64 half steps with the rest;
    # dweight: no lane of these tests adds more than 256 rows in a row
    return dx, 64 * F32 * size, (g * xhat).sum((0, 1)), 320 * F32 * terms


# --------------------------------------------------------------------------------- the cache
def quantise(x, store):
    """(values, scale): what the codes stand for, exactly; rows with an infinity or NaN are NaN."""
    wide = x.double()
    amax = wide.abs().amax(-1)
    fine = torch.isfinite(wide).all(-1)
    amax = torch.where(fine, amax, 1.0)
    if store == torch.int8:
        scale = torch.clamp((amax / 127).float().double(), min=2.0 ** -126)
        codes = torch.round(wide / scale[..., None])          # the quotient of 11 by 24 bits is never falsely a tie in 53
    else:
        scale = torch.full_like(amax, 2.0 ** -126)
        for e in range(-126, 128):                            # the least power of two that brings amax to 448
            scale = torch.where((448 * 2.0 ** (e - 1) < amax) & (amax <= 448 * 2.0 ** e), 2.0 ** e, scale)
        y = wide / scale[..., None]
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        codes = torch.round(y / step) * step
    nan = torch.where(fine, 0.0, float("nan"))
    return codes * scale[..., None] + nan[..., None], scale + nan


def values(cache, scale):
    """A cache's rows as the numbers that they stand for, in 64 bits."""
    if scale is None:
        return cache.double()
    return cache.float().double() * scale.double()[..., None]


def new_cache(pages, heads, page, columns, dtype, layout, device, fill=float("nan")):
    """(k, v, k_scale, v_scale) of one of three memory orders, all slots holding NaN: in 8 bits a NaN scale over arbitrary codes."""
    order = {"heads": (pages, 2, heads, page, columns), "tokens": (pages, page, 2, heads, columns),
             "apart": (2, pages, heads, page, columns)}[layout]
    both = torch.full(order, 85, dtype=torch.int8, device=device).view(dtype) if dtype in CODES else \
        torch.full(order, fill, dtype=dtype, device=device)
    scales = torch.full(order[:-1], fill, device=device) if dtype in CODES else None

    def split(t):
        if t is None:
            return None, None
        if layout == "heads":
            return t[:, 0], t[:, 1]
        if layout == "tokens":
            return t[:, :, 0].transpose(1, 2), t[:, :, 1].transpose(1, 2)
        return t[0], t[1]
    return *split(both), *split(scales)


# --------------------------------------------------------------------------------- attention
def attention(q, k_cache, v_cache, k_scale, v_scale, table, lengths, scale):
    """(out, its slack, lse, its slack), sequence by sequence in 64 bits."""
    batch, heads, columns = q.shape
    kv_heads, page = k_cache.shape[1], k_cache.shape[2]
    group = heads // kv_heads
    out = torch.zeros((batch, heads, columns), dtype=torch.float64, device=q.device)
    out_slack = torch.zeros_like(out)
    lse = torch.full((batch, heads), -float("inf"), dtype=torch.float64, device=q.device)
    lse_slack = torch.zeros_like(lse)
    for b in range(batch):
        length = min(max(int(lengths[b]), 0), table.shape[1] * page)
        if length == 0:
            continue
        pages = table[b, :-(-length // page)].long()
        good = (pages >= 0) & (pages < k_cache.shape[0])
        live = good.repeat_interleave(page)[:length]
        rows, sizes = [], []
        for cache, size in ((k_cache, k_scale), (v_cache, v_scale)):
            safe = torch.where(good, pages, 0)
            part = cache.view(torch.int8)[safe].view(cache.dtype) if cache.dtype in CODES else cache[safe]
            part = values(part, None if size is None else size[safe])
            row_size = torch.ones(part.shape[:3], dtype=torch.float64, device=q.device) if size is None else size[safe].double()
            sizes.append(row_size.permute(1, 0, 2).reshape(kv_heads, -1)[:, :length][:, live])
            rows.append(part.permute(1, 0, 2, 3).reshape(kv_heads, -1, columns)[:, :length][:, live])
        k, v = rows
        query = q[b].double().reshape(kv_heads, group, columns)
        scores = torch.einsum("hgd,hld->hgl", query, k) * scale
        size = torch.einsum("hgd,hld->hgl", query.abs(), k.abs()) * abs(scale)
        # a score's error: the products are exact, their sum adds columns terms in f32, its scaling five
        # more half steps (of the score in units of log2 e); 2^-21 is the relative error of exp2 and log2
        delta = (columns + 16) * F32 * size.amax(-1).nan_to_num(0, 0, 0) + 2.0 ** -20
        weights = torch.softmax(scores, -1)
        # the weights enter the second product with 16 bits or more, the sums add in f32 over
        # length / 64 steps and a fixed tree
        share = 2 * delta[..., None] + 2.0 ** -15 + (length / 64 + 64) * F32
        out[b] = torch.einsum("hgl,hld->hgd", weights, v).reshape(heads, columns)
        out_slack[b] = (share * torch.einsum("hgl,hld->hgd", weights, v.abs())).reshape(heads, columns)
        # As f16 (f16 and 8-bit caches) a weight is the sum of two halves relative to the largest weight so far, each
        # with the type's steps: the second half's are never finer than 2^-24, so a weight w_j (times its row's scale
        # z_j in 8 bits) is off by up to 2^-25 max(w z) however small it is, and a result by that times
        # sum |v_j| / z_j.  With bf16's exponents the floor is exp2's own, 2^-126.
        floor = 2.0 ** (-126 if k_cache.dtype == torch.bfloat16 else -25)
        largest = (weights * sizes[1][:, None, :]).amax(-1, keepdim=True)
        out_slack[b] += (floor * largest * (v.abs() / sizes[1][..., None]).sum(1)[:, None, :]).reshape(heads, columns)
        lse[b] = torch.logsumexp(scores, -1).reshape(-1)
        lse_slack[b] = (delta + (length / 64 + 64) * F32).reshape(-1) + 4 * F32 * lse[b].abs().nan_to_num(0, 0, 0)
    return out, out_slack.nan_to_num(0, 0, 0), lse, lse_slack
