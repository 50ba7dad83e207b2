"""What the operators around a key-value cache refuse, without a device: the C entries check every
argument before their first CUDA call, and ops checks types and shapes before that."""
import ctypes

import pytest
import torch

import plain_heads as plain
from intent_b200 import _native, ops

BASE = 1 << 20     # a 16-byte aligned address that nothing reads


def view(*shape, address=BASE, strides=None):
    if strides is None:
        strides, step = [], 1
        for extent in reversed(shape):
            strides.insert(0, step)
            step *= extent
    return [address, *shape, *strides]


def call(name, *parts):
    """The views among `parts` as one array of slots, then the rest."""
    slots = [x or 0 for part in parts if isinstance(part, list) for x in part]
    return _native.entry(name)((ctypes.c_int64 * len(slots))(*slots), len(slots), *(x for x in parts if not isinstance(x, list)))


SPACE = view(64, address=BASE + (1 << 40))
FAR = [BASE + (i << 34) for i in range(1, 12)]


def rotary(**change):
    p = {"q": view(5, 4, 64, address=FAR[0]), "k": view(5, 2, 64, address=FAR[1]), "qw": view(64), "kw": view(64),
         "cos": view(100, 32), "sin": view(100, 32), "positions": view(5), "qo": view(5, 4, 64, address=FAR[2]),
         "ko": view(5, 2, 64, address=FAR[3]), "epsilon": 1e-6, "space": SPACE, "dtype": 2, "interleaved": 0} | change
    return call("b200_head_norm_rotary", *p.values(), None)


@pytest.mark.parametrize("change, status", [
    ({"dtype": 3}, 1), ({"interleaved": 2}, 1), ({"epsilon": -1.0}, 1), ({"epsilon": float("nan")}, 1),
    ({"q": view(5, 4, 64, address=0)}, 1), ({"q": view(-5, 4, 64)}, 1), ({"q": view(6, 4, 64, address=FAR[0])}, 1),
    ({"k": view(5, 2, 80, address=FAR[1])}, 1), ({"qo": view(5, 3, 64, address=FAR[2])}, 1),
    ({"qw": view(32)}, 1), ({"kw": view(64, strides=[2])}, 2), ({"kw": view(64, address=BASE + 2)}, 2),
    ({"cos": view(99, 32)}, 1), ({"cos": view(100, 12), "sin": view(100, 12)}, 2), ({"cos": view(100, 40), "sin": view(100, 40)}, 2),
    ({"cos": view(100, 0), "sin": view(100, 0)}, 2), ({"cos": view(100, 32, strides=[33, 1])}, 2),
    ({"positions": view(4)}, 1), ({"positions": view(5, address=0)}, 1), ({"space": view(32)}, 1), ({"space": view(64, address=0)}, 1),
    ({"q": view(5, 4, 64, strides=[256, 64, 2], address=FAR[0])}, 2), ({"q": view(5, 4, 64, strides=[260, 64, 1], address=FAR[0])}, 2),
    ({"q": view(5, 4, 64, address=FAR[0] + 8)}, 2),
    ({"qo": view(5, 4, 64, address=FAR[0] + 128)}, 1),                        # half over its input
    ({"qo": view(5, 4, 64, address=FAR[1])}, 1),                              # on the other input
    ({"qo": view(5, 4, 64, address=FAR[3])}, 1),                              # on the other output
    ({"qo": view(5, 4, 64, address=FAR[2], strides=[0, 64, 1])}, 1),          # one row for all tokens
    ({"q": view(5, 4, 272, address=FAR[0]), "k": view(5, 2, 272, address=FAR[1]), "qo": view(5, 4, 272, address=FAR[2]),
      "ko": view(5, 2, 272, address=FAR[3]), "qw": view(272), "kw": view(272)}, 2),
    ({"q": view(5, 4, 64, strides=[1 << 62, 64, 1], address=FAR[0])}, 1),
])
def test_head_norm_rotary_refuses(change, status):
    assert rotary(**change) == status


def test_head_norm_rotary_of_nothing_is_done():
    nothing = {"q": view(0, 4, 64, address=0), "k": view(0, 2, 64, address=0), "qo": view(0, 4, 64, address=0),
               "ko": view(0, 2, 64, address=0), "positions": view(0, address=0)}
    assert rotary(**nothing) == 0


def test_rotary_views_of_one_projection_are_taken_apart():
    """q and k as slices of one tensor, written in place, pass the overlap checks (a launch without a
    device then fails as a CUDA error, not as a refusal)."""
    if torch.cuda.is_available():
        pytest.skip("would launch")
    q = view(5, 4, 64, strides=[512, 64, 1], address=FAR[0])
    k = view(5, 2, 64, strides=[512, 64, 1], address=FAR[0] + 4 * 64 * 2)
    assert rotary(q=q, k=k, qo=q, ko=k) == _native.ERR_CUDA
    k_over = view(5, 2, 64, strides=[512, 64, 1], address=FAR[0] + 3 * 64 * 2)
    assert rotary(q=q, k=k_over, qo=q, ko=k_over) == 1


def test_an_output_may_only_be_the_input_of_its_own_rows():
    """With as many key heads as query heads q's output could pass for k."""
    even = {"k": view(5, 4, 64, address=FAR[1]), "ko": view(5, 4, 64, address=FAR[3])}
    assert rotary(**even, qo=view(5, 4, 64, address=FAR[1])) == 1
    assert rotary(**(even | {"ko": view(5, 4, 64, address=FAR[0])})) == 1
    assert rotary(**(even | {"ko": view(5, 4, 64, address=FAR[2])})) == 1
    grads = {"k": view(5, 4, 64, address=FAR[1]), "gk": view(5, 4, 64, address=FAR[5]), "dk": view(5, 4, 64, address=FAR[3]),
             "partial": view(64, 64, address=FAR[8])}
    for place in (FAR[1], FAR[5], FAR[3]):
        assert backward(**grads, dq=view(5, 4, 64, address=place)) == 1
    if not torch.cuda.is_available():
        for place in (FAR[0], FAR[4]):
            assert backward(**grads, dq=view(5, 4, 64, address=place)) == _native.ERR_CUDA


def backward(**change):
    rows = ctypes.c_int64()
    assert _native.entry("b200_head_norm_rotary_scratch")(5, 4, 2, 64, ctypes.byref(rows)) == 0
    p = {"gq": view(5, 4, 64, address=FAR[4]), "gk": view(5, 2, 64, address=FAR[5]), "q": view(5, 4, 64, address=FAR[0]),
         "k": view(5, 2, 64, address=FAR[1]), "qw": view(64), "kw": view(64), "cos": view(100, 32), "sin": view(100, 32),
         "positions": view(5), "dq": view(5, 4, 64, address=FAR[2]), "dk": view(5, 2, 64, address=FAR[3]), "dqw": view(64, address=FAR[6]),
         "dkw": view(64, address=FAR[7]), "partial": view(rows.value, 64, address=FAR[8]), "epsilon": 1e-6, "space": SPACE,
         "dtype": 0, "interleaved": 1} | change
    return call("b200_head_norm_rotary_backward", *p.values(), None)


@pytest.mark.parametrize("change, status", [
    ({"gq": view(4, 4, 64, address=FAR[4])}, 1), ({"dqw": view(32)}, 1), ({"dkw": view(64, address=0)}, 1),
    ({"dqw": view(64, strides=[2])}, 2), ({"partial": view(0, 64)}, 1), ({"partial": view(9, 64, strides=[128, 1])}, 2),
    ({"dq": view(5, 4, 64, address=FAR[4] + 256)}, 1), ({"dq": view(5, 4, 64, address=FAR[5])}, 1), ({"dk": view(5, 2, 64, address=FAR[2])}, 1),
])
def test_head_norm_rotary_backward_refuses(change, status):
    assert backward(**change) == status


def write(name="b200_cache_write", **change):
    p = {"k": view(6, 2, 64, address=FAR[0]), "v": view(6, 2, 64, address=FAR[1]), "slots": view(6),
         "kc": view(3, 2, 16, 64, address=FAR[2]), "vc": view(3, 2, 16, 64, address=FAR[3]), "ks": view(3, 2, 16, address=FAR[4]),
         "vs": view(3, 2, 16, address=FAR[5]), "space": SPACE, "dtype": 1, "store": 3} | change
    if name == "b200_cache_write":
        order = ("k", "v", "slots", "kc", "vc", "ks", "vs", "space", "dtype", "store")
    else:
        order = ("kc", "vc", "slots", "ks", "vs", "k", "v", "space", "dtype", "store")
    return call(name, *(p[n] for n in order), None)


@pytest.mark.parametrize("name", ["b200_cache_write", "b200_cache_read"])
@pytest.mark.parametrize("change, status", [
    ({"dtype": 0}, 1), ({"dtype": 3}, 1), ({"store": 0}, 1), ({"store": 5}, 1), ({"store": 2}, 1),     # f16 rows, bf16 cache
    ({"k": view(6, 3, 64, address=FAR[0])}, 1), ({"k": view(6, 2, 48, address=FAR[0])}, 1), ({"v": view(5, 2, 64, address=FAR[1])}, 1),
    ({"slots": view(5)}, 1), ({"slots": view(6, address=0)}, 1), ({"slots": view(6, address=BASE + 4)}, 2),
    ({"vc": view(3, 2, 8, 64, address=FAR[3])}, 1), ({"kc": view(3, 2, 16, 64, address=0)}, 1),
    ({"kc": view(3, 2, 16, 64, address=FAR[2] + 8)}, 2), ({"kc": view(3, 2, 16, 64, address=FAR[2], strides=[2048, 1024, 72, 1])}, 2),
    ({"kc": view(3, 2, 16, 64, address=FAR[2], strides=[2048, 1024, 64, 2])}, 2),
    ({"ks": view(3, 2, 15, address=FAR[4])}, 1), ({"vs": view(3, 2, 16, address=0)}, 1), ({"vs": view(3, 2, 16, address=FAR[5] + 2)}, 2),
    ({"k": view(6, 2, 64, address=FAR[0], strides=[124, 64, 1])}, 2), ({"k": view(6, 2, 64, address=FAR[2])}, 1),
    ({"space": view(8)}, 1),
    ({"k": view(6, 2, 24, address=FAR[0]), "v": view(6, 2, 24, address=FAR[1]), "kc": view(3, 2, 16, 24, address=FAR[2]),
      "vc": view(3, 2, 16, 24, address=FAR[3])}, 2),
])
def test_cache_entries_refuse(name, change, status):
    assert write(name, **change) == status


def test_cache_write_refuses_what_overlaps_itself():
    assert write(vc=view(3, 2, 16, 64, address=FAR[2])) == 1
    assert write(vc=view(3, 2, 16, 64, address=FAR[2] + 1024)) == 1            # shifted by one head of the same pages
    assert write(kc=view(3, 2, 16, 64, address=FAR[2], strides=[0, 1024, 64, 1])) == 1
    assert write(vs=view(3, 2, 16, address=FAR[4])) == 1
    assert write("b200_cache_read", v=view(6, 2, 64, address=FAR[0])) == 1
    assert write("b200_cache_read", k=view(6, 2, 64, address=FAR[0], strides=[0, 64, 1])) == 1


def test_cache_halves_of_one_allocation_are_taken_apart():
    if torch.cuda.is_available():
        pytest.skip("would launch")
    for strides, shift in (([4096, 1024, 64, 1], 2048), ([4096, 64, 256, 1], 128)):   # (pages, 2, ...) and (pages, page, 2, ...)
        kc, vc = (view(3, 2, 16, 64, address=FAR[2] + at, strides=strides) for at in (0, shift))
        assert write(kc=kc, vc=vc) == _native.ERR_CUDA


def attend(**change):
    words = ctypes.c_int64()
    assert _native.entry("b200_paged_attention_scratch")(2, 8, 2, 64, 4800, 2, ctypes.byref(words)) == 0
    none3, none2 = [None] + [0] * 6, [None] + [0] * 4
    p = {"q": view(2, 8, 64, address=FAR[0]), "kc": view(9, 2, 16, 64, address=FAR[1]), "vc": view(9, 2, 16, 64, address=FAR[2]),
         "ks": none3, "vs": none3, "table": view(2, 300), "lengths": view(2), "out": view(2, 8, 64, address=FAR[3]), "lse": none2,
         "scale": 0.125, "partial": view(words.value, address=FAR[4]), "space": SPACE, "dtype": 2, "store": 2} | change
    return call("b200_paged_attention", *p.values(), None)


@pytest.mark.parametrize("change, status", [
    ({"dtype": 0}, 1), ({"store": 1}, 1), ({"store": 3}, 1), ({"q": view(2, 7, 64, address=FAR[0])}, 1),
    ({"q": view(2, 8, 32, address=FAR[0])}, 1), ({"out": view(2, 4, 64, address=FAR[3])}, 1), ({"out": view(2, 8, 64, address=FAR[0])}, 1),
    ({"out": view(2, 8, 64, address=FAR[3], strides=[0, 64, 1])}, 1), ({"table": view(3, 300)}, 1), ({"lengths": view(1)}, 1),
    ({"lengths": view(2, address=0)}, 1), ({"lse": view(2, 4, address=FAR[5])}, 1), ({"scale": float("inf")}, 1),
    ({"partial": view(16, address=FAR[4])}, 1), ({"partial": view(1 << 20, address=0)}, 1), ({"partial": view(1 << 22, address=FAR[4] + 4)}, 1),
    ({"space": view(3)}, 1), ({"q": view(2, 8, 64, address=FAR[0] + 2)}, 2),
    ({"table": view(2, 1 << 28)}, 2),
    ({"kc": view(9, 2, 16, 96, address=FAR[1]), "vc": view(9, 2, 16, 96, address=FAR[2]), "q": view(2, 8, 96, address=FAR[0]),
      "out": view(2, 8, 96, address=FAR[3])}, 2),
    ({"kc": view(9, 0, 16, 64, address=FAR[1]), "vc": view(9, 0, 16, 64, address=FAR[2])}, 1),
])
def test_paged_attention_refuses(change, status):
    assert attend(**change) == status


def test_paged_attention_of_no_sequences_is_done():
    assert attend(q=view(0, 8, 64), out=view(0, 8, 64), table=view(0, 3), lengths=view(0)) == 0


def test_a_wrong_number_of_slots_is_refused():
    for name, tail in (("b200_head_norm_rotary", (1e-6, 0, 0)), ("b200_head_norm_rotary_backward", (1e-6, 0, 0)), ("b200_cache_write", (1, 1)),
                       ("b200_cache_read", (1, 1)), ("b200_paged_attention", (1.0, 1, 1))):
        words = (ctypes.c_int64 * 200)()
        for address, count in ((words, 0), (words, 12), (words, 200), (None, 12), (None, 0)):
            assert _native.entry(name)(address, count, *tail, None) == 1


def test_scratch_entries_check_their_extents():
    words = ctypes.c_int64()
    size = _native.entry("b200_paged_attention_scratch")
    assert size(2, 8, 3, 64, 10, 2, ctypes.byref(words)) == 1 and size(2, 8, 0, 64, 10, 2, ctypes.byref(words)) == 1
    assert size(1 << 40, 8, 2, 64, 1 << 30, 2, ctypes.byref(words)) == 0 and 0 < words.value < 1 << 24
    assert size(1 << 40, 8, 2, 64, 10, 2, ctypes.byref(words)) == 0 and 0 < words.value < 1 << 24
    assert size(2, 8, 2, 64, 10, 2, ctypes.byref(words)) == 0 and words.value == 0     # nothing is cut
    assert _native.entry("b200_head_norm_rotary_scratch")(-1, 8, 2, 64, ctypes.byref(words)) == 1


def test_ops_check_before_any_call():
    q, k, w = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.zeros(64)
    with pytest.raises(ValueError, match="executes on cuda"):
        ops.head_norm_rotary(q, k, w, w, torch.zeros(9, 32), torch.zeros(9, 32), torch.zeros(3, dtype=torch.int32))
    cache = torch.zeros(2, 2, 16, 64, dtype=torch.int8)
    with pytest.raises(ValueError, match="executes on cuda"):
        ops.cache_write(k, k, torch.zeros(3, dtype=torch.int64), cache, cache)
    for wrong, message in (((cache, None, None, torch.half), "needs k_scale"), ((cache.half(), w, w, torch.half), "has no scales"),
                           ((cache.half(), None, None, torch.bfloat16), "k_cache must have dtype torch.bfloat16"),
                           ((cache.float(), None, None, None), "k_cache must be float16"), (([], None, None, None), "k_cache must be a torch.Tensor")):
        with pytest.raises((TypeError, ValueError), match=message):
            ops._cache_type(*wrong)


def test_a_view_that_is_not_what_it_should_be_is_named():
    """The native module finds it before any call, ops says what is wrong with it.  (On this machine every tensor is on the
    wrong device, so the module stops at the first view and the checks here are those of the message.)"""
    plan = ops._Plan("b200_cache_write", """
        first? f32 rows
        x x rows columns
        y f32 columns
        z= x rows""", "rows")
    t, column = torch.zeros(3, 4), torch.zeros(4)
    for bad, tensors, error, message in (
            (1, (None, t.long()[:2], column, ...), ValueError, r"x must have shape \(3, 4\), got \(2, 4\)"),
            (1, (None, [1.0], column, ...), TypeError, "x must be a torch.Tensor"), (1, (None, None, column, ...), TypeError, "x must be a torch.Tensor"),
            (1, (None, column, column, ...), ValueError, r"x is a \(rows, columns\) tensor, got \(4,\)"),
            (1, (None, t, column, ...), ValueError, "executes on cuda"), (0, (t, t, column, ...), ValueError, r"first is a \(rows,\) tensor")):
        with pytest.raises(error, match=message):
            plan._refuse(bad, 0, tensors, (3,))
        with pytest.raises(error):
            plan(0, tensors, (3,), None, 1, 1)
    for wrong in ((1, 0, [], (), (), None, 1, 1), (1, 0, (), (), None, 1), (1, 0, plan.views, (), (), None, 1, 1),
                  (1, 0, (), (), ("x",), None, 1, 1), (1, 0, (), (), (), "x", 1, 1)):
        with pytest.raises(TypeError):
            _native.binding().invoke(*wrong)


# ------------------------------------------------------- the plain forms hold what they are held to
def test_plain_quantisation_against_every_code():
    """The nearest of all codes, ties to the even one, by trying each of them."""
    torch.manual_seed(1)
    rows = (torch.randn(40, 16) * torch.exp(2 * torch.randn(40, 1))).half()
    rows[0], rows[1, 3], rows[2, 5], rows[3] = 0, float("inf"), float("nan"), rows[3] * 2.0 ** -14
    rows[4] = torch.arange(16) + 0.5
    rows[4, 0] = 127                                            # scale 1: every other entry is a tie
    for store in plain.CODES:
        every = torch.arange(-127, 128).double() if store == torch.int8 else \
            torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
        every = every[every.isfinite()]
        value, scale = plain.quantise(rows, store)
        for row in range(40):
            if not rows[row].isfinite().all():
                assert value[row].isnan().all() and scale[row].isnan()
                continue
            distance = (rows[row].double()[:, None] - every[None, :] * scale[row]).abs()
            best = distance.amin(1)
            assert torch.equal((rows[row].double() - value[row]).abs(), best)
            if store == torch.int8:
                ties = (distance == best[:, None]).sum(1) > 1
                assert ((value[row] / scale[row])[ties] % 2 == 0).all()


def test_plain_rotary_gradient_against_autograd_and_differences():
    torch.manual_seed(2)
    x, w = torch.randn(7, 3, 32, dtype=torch.float64, requires_grad=True), torch.rand(32, dtype=torch.float64, requires_grad=True)
    angle = torch.rand(20, 8, dtype=torch.float64) * 6
    cos, sin, positions = angle.cos(), angle.sin(), torch.tensor([0, 19, -1, 5, 20, 3, 3], dtype=torch.int32)
    grad = torch.randn(7, 3, 32, dtype=torch.float64)
    for interleaved in (False, True):
        def loss(x_, w_):
            return (plain.norm_rotary(x_, w_, cos, sin, positions, 1e-6, interleaved)[0] * grad).sum()
        auto = torch.autograd.grad(loss(x, w), (x, w))
        dx, _, dw, _ = plain.norm_rotary_backward(grad, x.detach(), w.detach(), cos, sin, positions, 1e-6, interleaved)
        assert (dx - auto[0]).abs().max() < 1e-12 and (dw - auto[1]).abs().max() < 1e-12
        assert not dx[2].any() and not dx[4].any()
        step, h = torch.randn_like(x), 1e-6
        slope = (loss(x + h * step, w) - loss(x - h * step, w)) / (2 * h)
        assert abs((slope - (dx * step).sum()).item()) < 1e-6 * (dx * step).abs().sum().item()
