"""Direct operator calls over CUDA ``torch`` tensors.

Each function packs its tensors into the flat slot list of the C ABI
(pointer, extents, element strides per view — the layout
``lib/Serialization/NativeABI.cpp:80-118`` defines), appends the private tail
and the current CUDA stream, and makes ONE foreign call.  Nothing here computes
on the host and nothing synchronises: like the reference's GPU launches the work
is enqueued on torch's current stream (``doc/getting-started/usage.en.md:53-55``).
Outputs are allocated the way the reference runtime allocates omitted ``Out``
buffers: contiguous ``torch.empty`` on the argument device
(``python/intent/runtime/torch_views.py:59-82``).
"""
from __future__ import annotations

import ctypes
from functools import lru_cache

import torch

from . import _native

_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int8: 3, torch.float8_e4m3fn: 4}


def _slots(tensor: torch.Tensor) -> list:
    return [tensor.data_ptr(), *tensor.shape, *tensor.stride()]


def _stream(tensor: torch.Tensor) -> int:
    return torch.cuda.current_stream(tensor.device).cuda_stream


def _require_cuda(*tensors: torch.Tensor) -> torch.device:
    device = tensors[0].device
    for tensor in tensors:
        if not isinstance(tensor, torch.Tensor):
            raise TypeError("intent_b200 operators take torch.Tensor arguments")
        if tensor.device.type != "cuda":
            raise ValueError(f"intent_b200 executes on cuda, but an argument is on {tensor.device}")
        if tensor.device != device:
            raise ValueError("arguments span different devices")
    return device


def _expect(name: str, tensor: torch.Tensor, dtype: torch.dtype, shape=None) -> None:
    """What the runtime binder checks for a bound view (``B200Program._observe``), for callers
    that come straight here: a wrong element type or extent must never reach the kernel, which
    trusts them (an int64 index array read as int32, or an output buffer of half the size, would
    send loads and stores out of bounds)."""
    if tensor.dtype != dtype:
        raise TypeError(f"{name} must have dtype {dtype}, got {tensor.dtype}")
    if shape is not None and tuple(tensor.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(tensor.shape)}")


def _float_type(name: str, tensor: torch.Tensor, allowed=(torch.float32, torch.float16, torch.bfloat16)) -> torch.dtype:
    if tensor.dtype not in allowed:
        raise TypeError(f"{name} must be one of {', '.join(str(d) for d in allowed)}, got {tensor.dtype}")
    return tensor.dtype


def _call(name: str, device: torch.device, *arguments) -> None:
    with torch.cuda.device(device):
        _native.check(name, _native.entry(name)(*arguments))


_workspaces: dict[torch.device, torch.Tensor] = {}


def workspace(device: torch.device) -> torch.Tensor:
    """The zero-initialised int32 status/workspace view the tensor-core entries take."""
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    if device not in _workspaces:
        _workspaces.setdefault(device, torch.zeros(_native.WORKSPACE_WORDS, dtype=torch.int32, device=device))
    return _workspaces[device]


def workspace_status(device: torch.device) -> None:
    """Synchronise and raise if a bounded device-side wait gave up."""
    ws = workspace(device)
    detail = ctypes.c_int32(0)
    with torch.cuda.device(ws.device):
        status = _native.entry("b200_workspace_status")(ws.data_ptr(), ctypes.byref(detail), _stream(ws))
    if status != _native.OK:
        ws.zero_()
    _native.check("b200_workspace_status", status)


def softmax(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    device = _require_cuda(x) if out is None else _require_cuda(x, out)
    _float_type("x", x)
    if x.dim() != 2:
        raise ValueError("softmax takes a matrix")
    y = torch.empty(x.shape, dtype=x.dtype, device=device) if out is None else out
    _expect("out", y, x.dtype, x.shape)
    _call("b200_softmax", device, *_slots(x), *_slots(y), _CODES[x.dtype], _stream(x))
    return y


def layer_norm(x, weight, bias, inverse_features: float, epsilon: float, out=None, *, centered=None):
    device = _require_cuda(x, weight, bias) if out is None else _require_cuda(x, weight, bias, out)
    _float_type("x", x)
    if x.dim() != 2:
        raise ValueError("layer_norm takes a matrix")
    _expect("weight", weight, x.dtype, (x.shape[1],))
    _expect("bias", bias, x.dtype, (x.shape[1],))
    y = torch.empty(x.shape, dtype=x.dtype, device=device) if out is None else out
    _expect("out", y, x.dtype, x.shape)
    if centered is None:  # the f32 kernel of the reference is the uncentred one
        centered = x.dtype != torch.float32
    _call("b200_layer_norm", device, *_slots(x), *_slots(weight), *_slots(bias), *_slots(y),
          float(inverse_features), float(epsilon), _CODES[x.dtype], int(centered), _stream(x))
    return y


def gemm(a, b, out=None, *, relu: bool = False):
    device = _require_cuda(a, b) if out is None else _require_cuda(a, b, out)
    _float_type("a", a, (torch.float16, torch.bfloat16))
    if a.dim() != 2 or b.dim() != 2:
        raise ValueError("gemm takes two matrices")
    _expect("b", b, a.dtype, (a.shape[1], b.shape[1]))
    c = torch.empty((a.shape[0], b.shape[1]), dtype=a.dtype, device=device) if out is None else out
    _expect("out", c, a.dtype, (a.shape[0], b.shape[1]))
    _call("b200_gemm", device, *_slots(a), *_slots(b), *_slots(c), *_slots(workspace(device)),
          _CODES[a.dtype], int(relu), _stream(a))
    return c


def flash_attention(q, k, v, scale: float, out=None, *, head_group: int = 1, causal: bool = True):
    device = _require_cuda(q, k, v) if out is None else _require_cuda(q, k, v, out)
    _float_type("q", q, (torch.float16, torch.bfloat16))
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("flash_attention takes (batch, heads, sequence, head_dim) tensors")
    _expect("k", k, q.dtype, (q.shape[0], k.shape[1], k.shape[2], q.shape[3]))
    _expect("v", v, q.dtype, (q.shape[0], k.shape[1], k.shape[2], v.shape[3]))
    if out is None:
        out = torch.empty((*q.shape[:3], v.shape[3]), dtype=q.dtype, device=device)
    _expect("out", out, q.dtype, (*q.shape[:3], v.shape[3]))
    _call("b200_flash_attention", device, *_slots(q), *_slots(k), *_slots(v), *_slots(out),
          float(scale), *_slots(workspace(device)), _CODES[q.dtype], int(head_group), int(causal),
          _stream(q))
    return out


def _csr_operands(row_offsets, column_indices, values) -> None:
    _expect("row_offsets", row_offsets, torch.int32)
    _expect("column_indices", column_indices, torch.int32)
    _expect("values", values, torch.float32, column_indices.shape)
    if row_offsets.dim() != 1 or column_indices.dim() != 1 or row_offsets.numel() < 1:
        raise ValueError("CSR arrays have one axis and row_offsets holds rows + 1 entries")


def csr_spmm(row_offsets, column_indices, values, dense, out=None, *, state=None):
    """`state`: the call's int32 workspace (``workspace(device)`` by default); calls that may overlap
    on different streams need one each."""
    device = _require_cuda(row_offsets, column_indices, values, dense, *(() if out is None else (out,)))
    _csr_operands(row_offsets, column_indices, values)
    if dense.dim() != 2:
        raise ValueError("dense must be a matrix")
    _expect("dense", dense, torch.float32)
    if out is None:
        out = torch.empty((row_offsets.numel() - 1, dense.shape[1]), dtype=torch.float32, device=device)
    _expect("out", out, torch.float32, (row_offsets.numel() - 1, dense.shape[1]))
    if state is not None:
        _expect("state", state, torch.int32)
    _call("b200_csr_spmm", device, *_slots(row_offsets), *_slots(column_indices), *_slots(values),
          *_slots(dense), *_slots(out), *_slots(workspace(device) if state is None else state), _stream(dense))
    return out


def csr_spmv(row_offsets, column_indices, values, vector, out=None):
    device = _require_cuda(row_offsets, column_indices, values, vector, *(() if out is None else (out,)))
    _csr_operands(row_offsets, column_indices, values)
    _expect("vector", vector, torch.float32)
    if vector.dim() != 1:
        raise ValueError("vector must have one axis")
    if out is None:
        out = torch.empty((row_offsets.numel() - 1,), dtype=torch.float32, device=device)
    _expect("out", out, torch.float32, (row_offsets.numel() - 1,))
    _call("b200_csr_spmv", device, *_slots(row_offsets), *_slots(column_indices), *_slots(values),
          *_slots(vector), *_slots(out), _stream(vector))
    return out


def softmax_backward(probabilities, upstream, out=None):
    device = _require_cuda(probabilities, upstream, *(() if out is None else (out,)))
    _expect("probabilities", probabilities, torch.float32)
    _expect("upstream", upstream, torch.float32, probabilities.shape)
    if out is None:
        out = torch.empty(probabilities.shape, dtype=probabilities.dtype, device=device)
    _expect("out", out, torch.float32, probabilities.shape)
    _call("b200_softmax_backward", device, *_slots(probabilities), *_slots(upstream), *_slots(out),
          _CODES[probabilities.dtype], _stream(probabilities))
    return out


def layer_norm_backward_rows(x, dy, weight, mean, rstd, dw_partial, db_partial, inverse_features: float, out=None):
    """Returns dx; accumulates into ``dw_partial`` / ``db_partial`` (InOut) in place."""
    device = _require_cuda(x, dy, weight, mean, rstd, dw_partial, db_partial, *(() if out is None else (out,)))
    _expect("x", x, torch.bfloat16)
    if x.dim() != 2 or dw_partial.dim() != 2:
        raise ValueError("layer_norm_backward_rows takes matrices")
    _expect("dy", dy, torch.bfloat16, x.shape)
    _expect("weight", weight, torch.bfloat16, (x.shape[1],))
    _expect("mean", mean, torch.float32, (x.shape[0],))
    _expect("rstd", rstd, torch.float32, (x.shape[0],))
    _expect("dw_partial", dw_partial, torch.bfloat16, (dw_partial.shape[0], x.shape[1]))
    _expect("db_partial", db_partial, torch.bfloat16, dw_partial.shape)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=device)
    _expect("out", out, torch.bfloat16, x.shape)
    _call("b200_layer_norm_backward_rows", device, *_slots(x), *_slots(dy), *_slots(weight), *_slots(mean),
          *_slots(rstd), *_slots(out), *_slots(dw_partial), *_slots(db_partial), float(inverse_features), _stream(x))
    return out


def layer_norm_backward_reduce(dw_partial, db_partial, dw=None, db=None):
    device = _require_cuda(dw_partial, db_partial, *(t for t in (dw, db) if t is not None))
    _expect("dw_partial", dw_partial, torch.bfloat16)
    if dw_partial.dim() != 2:
        raise ValueError("the partial sums are matrices")
    _expect("db_partial", db_partial, torch.bfloat16, dw_partial.shape)
    columns = dw_partial.shape[1]
    for name, tensor in (("dw", dw), ("db", db)):
        if tensor is not None:
            _expect(name, tensor, torch.float32, (columns,))
    if dw is None:
        dw = torch.empty((columns,), dtype=torch.float32, device=device)
    if db is None:
        db = torch.empty((columns,), dtype=torch.float32, device=device)
    _call("b200_layer_norm_backward_reduce", device, *_slots(dw_partial), *_slots(db_partial), *_slots(dw), *_slots(db),
          _stream(dw_partial))
    return dw, db


def attention_backward_delta(output, grad_output, out=None):
    device = _require_cuda(output, grad_output, *(() if out is None else (out,)))
    _float_type("output", output, (torch.float16, torch.bfloat16))
    if output.dim() != 4:
        raise ValueError("attention_backward_delta takes (batch, heads, sequence, head_dim) tensors")
    _expect("grad_output", grad_output, output.dtype, output.shape)
    if out is None:
        out = torch.empty(output.shape[:3], dtype=torch.float32, device=device)
    _expect("out", out, torch.float32, output.shape[:3])
    _call("b200_attention_backward_delta", device, *_slots(output), *_slots(grad_output), *_slots(out),
          _CODES[output.dtype], _stream(output))
    return out


def _attention_backward_operands(q, k, v, grad_output, lse, delta) -> None:
    _float_type("q", q, (torch.float16, torch.bfloat16))
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("attention backward takes (batch, heads, sequence, head_dim) tensors")
    _expect("k", k, q.dtype, (q.shape[0], k.shape[1], k.shape[2], q.shape[3]))
    _expect("v", v, q.dtype, k.shape)
    _expect("grad_output", grad_output, q.dtype, q.shape)
    _expect("lse", lse, torch.float32, q.shape[:3])
    _expect("delta", delta, torch.float32, q.shape[:3])


def attention_backward_dkdv(q, k, v, grad_output, lse, delta, scale: float, *, head_group: int = 1,
                            causal: bool = True, grad_k=None, grad_v=None):
    device = _require_cuda(q, k, v, grad_output, lse, delta, *(t for t in (grad_k, grad_v) if t is not None))
    _attention_backward_operands(q, k, v, grad_output, lse, delta)
    grad_k = torch.empty(k.shape, dtype=k.dtype, device=device) if grad_k is None else grad_k
    grad_v = torch.empty(v.shape, dtype=v.dtype, device=device) if grad_v is None else grad_v
    _expect("grad_k", grad_k, q.dtype, k.shape)
    _expect("grad_v", grad_v, q.dtype, v.shape)
    space = workspace(device)
    _call("b200_attention_backward_dkdv", device, *_slots(q), *_slots(k), *_slots(v), *_slots(grad_output),
          *_slots(lse), *_slots(delta), *_slots(grad_k), *_slots(grad_v), float(scale), *_slots(space),
          _CODES[q.dtype], int(head_group), int(causal), _stream(q))
    return grad_k, grad_v


def attention_backward_dq(q, k, v, grad_output, lse, delta, scale: float, *, head_group: int = 1,
                          causal: bool = True, grad_q=None):
    device = _require_cuda(q, k, v, grad_output, lse, delta, *(() if grad_q is None else (grad_q,)))
    _attention_backward_operands(q, k, v, grad_output, lse, delta)
    grad_q = torch.empty(q.shape, dtype=q.dtype, device=device) if grad_q is None else grad_q
    _expect("grad_q", grad_q, q.dtype, q.shape)
    space = workspace(device)
    _call("b200_attention_backward_dq", device, *_slots(q), *_slots(k), *_slots(v), *_slots(grad_output),
          *_slots(lse), *_slots(delta), *_slots(grad_q), float(scale), *_slots(space), _CODES[q.dtype],
          int(head_group), int(causal), _stream(q))
    return grad_q


# ---- operators around a key-value cache ------------------------------------------------------
# Calls of a few microseconds on the device, so their views are not packed here but by a native module.

def _cuda_device(tensor) -> int:
    """Index of the device that the call runs on, from its first tensor."""
    if not isinstance(tensor, torch.Tensor):
        raise TypeError("intent_b200 operators take torch.Tensor arguments")
    if not tensor.is_cuda:
        raise ValueError(f"intent_b200 executes on cuda, but an argument is on {tensor.device}")
    return tensor.get_device()


_addresses: dict[str, int] = {}
_native_invoke = None


def _invoke(name: str, device: int, views: tuple, number, code: int, other: int) -> tuple:
    """Calls an entry that takes its views as one array of slots, and returns the tensors that were made for it.
    ``views``: (name, tensor, dtype, shape), with ``...`` for the tensor if it is to be made, (name, ..., dtype, shape,
    True) for scratch, (name, None, rank) for a view that is not there; ``number``: the entry's f32 argument, if it
    has one.  Everything made is a contiguous allocation of the call's own in the current stream's order, so
    calls may overlap."""
    global _native_invoke
    entry = _addresses.get(name)
    if entry is None:
        _native_invoke = _native.binding().invoke
        entry = _addresses[name] = _native.address(name)
    made = _native_invoke(entry, device, views, number, code, other)
    if type(made) is not tuple:
        if made < 0:
            _refuse(views[-1 - made], device)
        _native.check(name, made)
    return made


def _refuse(view: tuple, device: int) -> None:
    """Raises what is wrong with a view."""
    name, tensor, dtype, shape = view
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    _expect(name, tensor, dtype, shape)
    if _cuda_device(tensor) != device:
        raise ValueError("arguments span different devices")
    raise ValueError(f"{name} must be a strided tensor")


def _outputs(made: tuple, *given) -> tuple:
    """The outputs of a call: those that the caller gave, and for the others what was made, in order."""
    rest = iter(made)
    return tuple(next(rest) if tensor is None else tensor for tensor in given)


_status_spaces: dict[int, tuple] = {}


def _status(device: int) -> tuple:
    """The view of ``workspace(device)``, where an entry records a bad index.  It is made once per device and
    shared by all streams, so the first call may not fall into a graph capture, whose replays would
    clear it, and its zeros have to be there before any other stream writes to it."""
    view = _status_spaces.get(device)
    if view is None:
        where = torch.device("cuda", device)
        with torch.cuda.device(where):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("call this operator once outside a graph capture before capturing it")
            space = workspace(where)
            torch.cuda.current_stream(where).synchronize()
        view = _status_spaces[device] = ("workspace", space, torch.int32, (_native.WORKSPACE_WORDS,))
    return view


@lru_cache(maxsize=4096)
def _scratch_size(name: str, device: int, *arguments) -> int:
    size = ctypes.c_int64(0)
    _call(name, torch.device("cuda", device), *arguments, ctypes.byref(size))
    return size.value


def _shape(name: str, tensor, rank: int, axes: str) -> tuple:
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if tensor.dim() != rank:
        raise ValueError(f"{name} is a {axes} tensor, got {tuple(tensor.shape)}")
    return tuple(tensor.shape)


def _rotary_shapes(q, k, cos) -> tuple:
    shape = _shape("q", q, 3, "(tokens, heads, head_dim)")
    k_shape = (shape[0], _shape("k", k, 3, "(tokens, heads, head_dim)")[1], shape[2])
    _float_type("q", q)
    return shape, k_shape, _shape("cos", cos, 2, "(rows, pairs)")


def head_norm_rotary(q, k, q_weight, k_weight, cos, sin, positions, epsilon: float = 1e-6, *, interleaved: bool = False,
                     q_out=None, k_out=None):
    """RMS norm of every head of ``q`` and ``k`` (tokens, heads, head_dim), times its weight, and the
    rotation by the token's position, in one launch.  ``cos`` and ``sin`` (rows, pairs) are f32 tables
    over positions; pair ``i`` is columns ``(i, i + pairs)``, or ``(2i, 2i + 1)`` with ``interleaved``, and
    columns from ``2 * pairs`` on are not turned.  ``positions`` (tokens,) int32: a negative one marks
    padding, whose rows become zeros; one behind the tables gives zeros too and is reported by
    ``workspace_status``.  Returns ``(q_out, k_out)``; an output may be its input."""
    device = _cuda_device(q)
    shape, k_shape, table = _rotary_shapes(q, k, cos)
    dtype, columns = q.dtype, shape[2:]
    made = _invoke(
        "b200_head_norm_rotary", device,
        (("q", q, dtype, shape), ("k", k, dtype, k_shape), ("q_weight", q_weight, dtype, columns),
         ("k_weight", k_weight, dtype, columns), ("cos", cos, torch.float32, table), ("sin", sin, torch.float32, table),
         ("positions", positions, torch.int32, shape[:1]), ("q_out", ... if q_out is None else q_out, dtype, shape),
         ("k_out", ... if k_out is None else k_out, dtype, k_shape), _status(device)), float(epsilon), _CODES[dtype], bool(interleaved))
    return _outputs(made, q_out, k_out)


def head_norm_rotary_backward(grad_q, grad_k, q, k, q_weight, k_weight, cos, sin, positions, epsilon: float = 1e-6, *,
                              interleaved: bool = False, dq=None, dk=None):
    """The gradients of ``head_norm_rotary``'s inputs from those of its outputs: ``(dq, dk, dq_weight,
    dk_weight)``, the weights' in f32.  Rows of padding get zeros and add nothing.  ``dq`` may be
    ``grad_q`` or ``q``, and ``dk`` likewise."""
    device = _cuda_device(q)
    shape, k_shape, table = _rotary_shapes(q, k, cos)
    dtype, columns = q.dtype, shape[2:]
    rows = _scratch_size("b200_head_norm_rotary_scratch", device, shape[0], shape[1], k_shape[1], shape[2])
    made = _invoke(
        "b200_head_norm_rotary_backward", device,
        (("grad_q", grad_q, dtype, shape), ("grad_k", grad_k, dtype, k_shape), ("q", q, dtype, shape), ("k", k, dtype, k_shape),
         ("q_weight", q_weight, dtype, columns), ("k_weight", k_weight, dtype, columns), ("cos", cos, torch.float32, table),
         ("sin", sin, torch.float32, table), ("positions", positions, torch.int32, shape[:1]),
         ("dq", ... if dq is None else dq, dtype, shape), ("dk", ... if dk is None else dk, dtype, k_shape),
         ("dq_weight", ..., torch.float32, columns), ("dk_weight", ..., torch.float32, columns), ("partial", ..., torch.float32, (rows, shape[2]), True),
         _status(device)), float(epsilon), _CODES[dtype], bool(interleaved))
    return _outputs(made, dq, dk, None, None)


_NO_SCALES = (("k_scale", None, 3), ("v_scale", None, 3))
_CACHE_TYPES = (torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn)


def _cache_views(k_cache, v_cache, k_scale, v_scale) -> tuple:
    """Shape of a paged cache, its views and its scales' views."""
    shape = _shape("k_cache", k_cache, 4, "(pages, heads, page_size, head_dim)")
    dtype = k_cache.dtype
    if dtype not in _CACHE_TYPES:
        raise TypeError(f"k_cache must be float16, bfloat16, int8 or float8_e4m3fn, got {dtype}")
    views = (("k_cache", k_cache, dtype, shape), ("v_cache", v_cache, dtype, shape))
    if dtype is torch.float16 or dtype is torch.bfloat16:
        if k_scale is not None or v_scale is not None:
            raise ValueError("a 16-bit cache has no scales")
        return shape, views, _NO_SCALES
    if k_scale is None or v_scale is None:
        raise ValueError("an 8-bit cache needs k_scale and v_scale")
    return shape, views, (("k_scale", k_scale, torch.float32, shape[:3]), ("v_scale", v_scale, torch.float32, shape[:3]))


def cache_write(k, v, slots, k_cache, v_cache, k_scale=None, v_scale=None):
    """Puts rows of keys and values (tokens, heads, head_dim), f16 or bf16, into the slots of a paged cache
    (pages, heads, page_size, head_dim) of any memory order with a unit inner stride, in one launch;
    slot = page * page_size + place, int64.  A cache of the rows' type gets them as they are.  One of int8 or
    float8_e4m3fn gets codes, and ``k_scale`` / ``v_scale`` (pages, heads, page_size) f32 a scale for each row:
    the largest magnitude / 127, or the power of two that brings it to at most 448; code * scale is the value.
    A row with an infinity or a NaN reads back as NaN throughout.  Negative slots mark padding and are
    skipped; so are slots behind the cache, which ``workspace_status`` reports.  The slots of one call that are not
    negative must differ.  Returns ``(k_cache, v_cache)``."""
    device = _cuda_device(k)
    dtype = _float_type("k", k, (torch.float16, torch.bfloat16))
    cache, views, scales = _cache_views(k_cache, v_cache, k_scale, v_scale)
    if k_cache.dtype is not dtype and k_cache.element_size() == 2:
        raise TypeError(f"k_cache must have dtype {dtype}, torch.int8 or torch.float8_e4m3fn, got {k_cache.dtype}")
    shape = (_shape("k", k, 3, "(tokens, heads, head_dim)")[0], cache[1], cache[3])
    _invoke("b200_cache_write", device,
            (("k", k, dtype, shape), ("v", v, dtype, shape), ("slots", slots, torch.int64, shape[:1]), *views, *scales,
             _status(device)), None, _CODES[dtype], _CODES[k_cache.dtype])
    return k_cache, v_cache


def cache_read(k_cache, v_cache, slots, k_scale=None, v_scale=None, *, dtype=None, k_out=None, v_out=None):
    """The rows of ``slots`` out of a cache that ``cache_write`` filled, ``(k, v)`` of shape (tokens, heads,
    head_dim): of a 16-bit cache as they are, of an 8-bit one as code * scale in ``dtype`` (f16 or bf16, the
    default).  Negative slots give zeros, and so do slots behind the cache, which ``workspace_status`` reports."""
    device = _cuda_device(k_cache)
    cache, views, scales = _cache_views(k_cache, v_cache, k_scale, v_scale)
    wide = k_cache.element_size() == 2
    if dtype is None:
        dtype = k_cache.dtype if wide else torch.bfloat16 if k_out is None else k_out.dtype
    if dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"dtype must be torch.float16 or torch.bfloat16, got {dtype}")
    if wide and dtype != k_cache.dtype:
        raise TypeError(f"a {k_cache.dtype} cache gives its rows as they are, not as {dtype}")
    shape = (_shape("slots", slots, 1, "(tokens,)")[0], cache[1], cache[3])
    made = _invoke(
        "b200_cache_read", device,
        (*views, ("slots", slots, torch.int64, shape[:1]), *scales, ("k_out", ... if k_out is None else k_out, dtype, shape),
         ("v_out", ... if v_out is None else v_out, dtype, shape), _status(device)), None, _CODES[dtype], _CODES[k_cache.dtype])
    return _outputs(made, k_out, v_out)


def paged_attention(q, k_cache, v_cache, block_table, lengths, scale: float, *, k_scale=None, v_scale=None, out=None,
                    return_lse: bool = False):
    """Attention of one new token a sequence: ``q`` (batch, heads, head_dim) over the first ``lengths[b]`` rows of
    each sequence in a paged cache (``cache_write``), whose pages row ``b`` of ``block_table`` (batch, columns)
    names in order; both int32.  heads is a multiple of the cache's heads, neighbouring query heads share a key
    head; head_dim is 64 or 128.  A sequence of length 0 gets zeros (and lse -infinity).  What lies behind a
    sequence, in its last page or in the table, is never used.  A page outside the cache is left out, a length
    past the table is cut there, and ``workspace_status`` reports both.  Returns ``out``, or ``(out, lse)``
    with the natural logarithm of the sums (f32)."""
    device = _cuda_device(q)
    dtype = _float_type("q", q, (torch.float16, torch.bfloat16))
    shape = _shape("q", q, 3, "(batch, heads, head_dim)")
    cache, views, scales = _cache_views(k_cache, v_cache, k_scale, v_scale)
    if k_cache.dtype is not dtype and k_cache.element_size() == 2:
        raise TypeError(f"k_cache must have dtype {dtype}, torch.int8 or torch.float8_e4m3fn, got {k_cache.dtype}")
    batch, heads, columns = shape
    if columns != cache[3]:
        raise ValueError(f"q has head_dim {columns}, the cache {cache[3]}")
    if cache[1] < 1 or heads < 1 or heads % cache[1]:
        raise ValueError(f"{heads} query heads are not a multiple of the cache's {cache[1]}")
    table = (batch, _shape("block_table", block_table, 2, "(batch, columns)")[1])
    store = _CODES[k_cache.dtype]
    words = _scratch_size("b200_paged_attention_scratch", device, batch, heads, cache[1], columns, table[1] * cache[2], store)
    made = _invoke(
        "b200_paged_attention", device,
        (("q", q, dtype, shape), *views, *scales, ("block_table", block_table, torch.int32, table),
         ("lengths", lengths, torch.int32, shape[:1]), ("out", ... if out is None else out, dtype, shape),
         ("lse", ..., torch.float32, shape[:2]) if return_lse else ("lse", None, 2),
         ("partial", ..., torch.float32, (words,), True), _status(device)), float(scale), _CODES[dtype], store)
    return _outputs(made, out, None) if return_lse else out if out is not None else made[0]


def gather_probe(table: torch.Tensor, gathers: int, *, variant: int = 1, hints: bool = True) -> None:
    """Enqueues the gather-rate probe over `table` (rows of 128 f32)."""
    device = _require_cuda(table)
    if table.dtype != torch.float32 or table.dim() != 2 or table.shape[1] != 128 or not table.is_contiguous():
        raise ValueError("gather_probe takes a contiguous f32 table of 128 columns")
    sink = _probe_sinks.get(device)
    if sink is None:
        sink = _probe_sinks[device] = torch.zeros(148 * 64 * 128 * 4, dtype=torch.float32, device=device)
    _call("b200_gather_probe", device, table.data_ptr(), table.shape[0], int(gathers), int(variant), int(hints),
          sink.data_ptr(), workspace(device).data_ptr(), _stream(table))


_probe_sinks: dict[torch.device, torch.Tensor] = {}


def csr_validate(row_offsets, column_indices, columns: int) -> None:
    device = _require_cuda(row_offsets, column_indices)
    where = ctypes.c_int64(-1)
    _call("b200_csr_validate", device, row_offsets.data_ptr(), row_offsets.numel() - 1,
          column_indices.data_ptr(), column_indices.numel(), int(columns), ctypes.byref(where),
          _stream(row_offsets))
