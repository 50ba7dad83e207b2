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
from threading import Lock

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
_workspaces_lock = Lock()


def workspace(device: torch.device) -> torch.Tensor:
    """The zero-initialised int32 status/workspace view that entries report to, one per device and shared by all
    streams.  Its zeros are there before anything else sees it, and it belongs to no graph: replays of one would
    clear its reports."""
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    space = _workspaces.get(device)
    if space is None:
        with _workspaces_lock:
            space = _workspaces.get(device)
            if space is None:
                space = _workspaces[device] = _zeroed(device)
    return space


def _zeroed(device: torch.device) -> torch.Tensor:
    if device.type != "cuda":
        return torch.zeros(_native.WORKSPACE_WORDS, dtype=torch.int32, device=device)
    with torch.cuda.device(device), torch.inference_mode(False):   # what is made in that mode cannot be cleared outside of it
        if torch.cuda.is_current_stream_capturing():
            return _native.binding().zeroed(device.index, _native.WORKSPACE_WORDS)
        space = torch.zeros(_native.WORKSPACE_WORDS, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()
        return space


def workspace_status(device: torch.device) -> None:
    """Synchronise and raise if a bounded device-side wait gave up (``NativeCallError``), or else if a position, slot,
    page or length was outside its table or cache (``ValueError``).  What was raised is cleared."""
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
# Calls of a few microseconds on the device, so their views are not checked and packed here but by a
# native module, after a plan.

_GIVEN, _OUTPUT, _SCRATCH, _OPTIONAL = range(4)


class _Plan:
    """The views of an entry that takes them as one array of slots, in its order.  ``views``: a line for each,
    "name dtype axis axis ...", where dtype x is the call's own, and axes of one name have one extent.  A name that
    ends in ``=`` is an output, in ``~`` scratch, in ``?`` a view that may be missing.  ``given``: the axes whose
    extents a call passes."""

    def __init__(self, entry: str, views: str, given: str = ""):
        self.entry, self.address = entry, None
        axes = {name: i for i, name in enumerate(given.split())}
        types = {"x": None, "f32": torch.float32, "i32": torch.int32, "i64": torch.int64}
        plan = []
        for line in views.strip().splitlines():
            name, dtype, *shape = line.split()
            kind = {"=": _OUTPUT, "~": _SCRATCH, "?": _OPTIONAL}.get(name[-1], _GIVEN)
            symbols = tuple(axes.setdefault(axis, len(axes)) for axis in shape)
            plan.append((name.rstrip("=~?"), types.get(dtype, dtype), symbols, kind))
        self.views, self.axes = tuple(plan), tuple(axes)

    def typed(self, **types):
        """The same plan with types in the place of names."""
        plan = _Plan.__new__(_Plan)
        plan.entry, plan.address, plan.axes = self.entry, None, self.axes
        plan.views = tuple((name, types.get(dtype, dtype) if isinstance(dtype, str) else dtype, *rest)
                           for name, dtype, *rest in self.views)
        return plan

    def __call__(self, device: int, tensors: tuple, extents: tuple, number, code: int, other: int) -> tuple:
        """Calls the entry on the current stream and returns the tensors that were made for it: those given as
        ``...``.  They, and the scratch, are contiguous allocations of the call's own in the stream's order, so
        calls may overlap."""
        if self.address is None:
            self.invoke, self.address = _native.binding().invoke, _native.address(self.entry)
        made = self.invoke(self.address, device, self.views, tensors, extents, number, code, other)
        if type(made) is not tuple:
            if made < 0:
                self._refuse(-1 - made, device, tensors, extents)
            _native.check(self.entry, made)
        return made

    def _refuse(self, bad: int, device: int, tensors: tuple, extents: tuple) -> None:
        """Raises what is wrong with a view, given that those before it are right."""
        known, call_type = dict(enumerate(extents)), None
        for (name, dtype, symbols, _), tensor in zip(self.views[:bad + 1], tensors):
            if tensor is ... or tensor is None and name != self.views[bad][0]:
                continue
            if not isinstance(tensor, torch.Tensor):
                raise TypeError(f"{name} must be a torch.Tensor")
            if tensor.dim() != len(symbols):
                axes = ", ".join(self.axes[symbol] for symbol in symbols)
                raise ValueError(f"{name} is a ({axes}{',' * (len(symbols) == 1)}) tensor, got {tuple(tensor.shape)}")
            call_type = tensor.dtype if dtype is None and call_type is None else call_type
            shape = tuple(known.setdefault(symbol, extent) for symbol, extent in zip(symbols, tensor.shape))
            _expect(name, tensor, call_type if dtype is None else dtype, shape)
            if _cuda_device(tensor) != device:
                raise ValueError("arguments span different devices")
        raise ValueError(f"{self.views[bad][0]} must be a strided tensor")


def _cuda_device(tensor) -> int:
    """Index of the device that the call runs on, from its first tensor."""
    if not isinstance(tensor, torch.Tensor):
        raise TypeError("intent_b200 operators take torch.Tensor arguments")
    if not tensor.is_cuda:
        raise ValueError(f"intent_b200 executes on cuda, but an argument is on {tensor.device}")
    return tensor.get_device()


def _outputs(made: tuple, *given) -> tuple:
    """The outputs of a call: those that the caller gave, and for the others what was made, in order."""
    rest = iter(made)
    return tuple(next(rest) if tensor is None else tensor for tensor in given)


_status_spaces: dict[int, torch.Tensor] = {}


def _status(device: int) -> torch.Tensor:
    """``workspace(device)``, where an entry records a bad index, by the device's number (a lookup takes a tenth of the time)."""
    space = _status_spaces.get(device)
    if space is None:
        space = _status_spaces[device] = workspace(torch.device("cuda", device))
    return space


@lru_cache(maxsize=4096)
def _scratch_size(name: str, device: int, *arguments) -> int:
    size = ctypes.c_int64(0)
    _call(name, torch.device("cuda", device), *arguments, ctypes.byref(size))
    return size.value


_ROTARY = _Plan("b200_head_norm_rotary", """
    q x tokens heads head_dim
    k x tokens kv_heads head_dim
    q_weight x head_dim
    k_weight x head_dim
    cos f32 rows pairs
    sin f32 rows pairs
    positions i32 tokens
    q_out= x tokens heads head_dim
    k_out= x tokens kv_heads head_dim
    workspace i32 words""")

_ROTARY_BACKWARD = _Plan("b200_head_norm_rotary_backward", """
    grad_q x tokens heads head_dim
    grad_k x tokens kv_heads head_dim
    q x tokens heads head_dim
    k x tokens kv_heads head_dim
    q_weight x head_dim
    k_weight x head_dim
    cos f32 rows pairs
    sin f32 rows pairs
    positions i32 tokens
    dq= x tokens heads head_dim
    dk= x tokens kv_heads head_dim
    dq_weight= f32 head_dim
    dk_weight= f32 head_dim
    partial~ f32 partial_rows head_dim
    workspace i32 words""", "partial_rows")


def head_norm_rotary(q, k, q_weight, k_weight, cos, sin, positions, epsilon: float = 1e-6, *, interleaved: bool = False,
                     q_out=None, k_out=None):
    """RMS norm of every head of ``q`` and ``k`` (tokens, heads, head_dim), times its weight, and the
    rotation by the token's position, in one launch.  ``cos`` and ``sin`` (rows, pairs) are f32 tables
    over positions; pair ``i`` is columns ``(i, i + pairs)``, or ``(2i, 2i + 1)`` with ``interleaved``, and
    columns from ``2 * pairs`` on are not turned.  ``positions`` (tokens,) int32: a negative one marks
    padding, whose rows become zeros; one behind the tables gives zeros too and is reported by
    ``workspace_status``.  Returns ``(q_out, k_out)``; an output may be its input."""
    device = _cuda_device(q)
    made = _ROTARY(device, (q, k, q_weight, k_weight, cos, sin, positions, ... if q_out is None else q_out,
                            ... if k_out is None else k_out, _status(device)),
                   (), float(epsilon), _CODES[_float_type("q", q)], bool(interleaved))
    return made if len(made) == 2 else _outputs(made, q_out, k_out)


def head_norm_rotary_backward(grad_q, grad_k, q, k, q_weight, k_weight, cos, sin, positions, epsilon: float = 1e-6, *,
                              interleaved: bool = False, dq=None, dk=None):
    """The gradients of ``head_norm_rotary``'s inputs from those of its outputs: ``(dq, dk, dq_weight,
    dk_weight)``, the weights' in f32.  Rows of padding get zeros and add nothing.  ``dq`` may be
    ``grad_q`` or ``q``, and ``dk`` likewise."""
    device = _cuda_device(q)
    if q.dim() != 3 or not isinstance(k, torch.Tensor) or k.dim() != 3:
        raise ValueError("q and k are (tokens, heads, head_dim) tensors")
    tokens, heads, head_dim = q.shape
    rows = _scratch_size("b200_head_norm_rotary_scratch", device, tokens, heads, k.shape[1], head_dim)
    made = _ROTARY_BACKWARD(device, (grad_q, grad_k, q, k, q_weight, k_weight, cos, sin, positions,
                                     ... if dq is None else dq, ... if dk is None else dk, ..., ..., ...,
                                     _status(device)),
                            (rows,), float(epsilon), _CODES[_float_type("q", q)], bool(interleaved))
    return made if len(made) == 4 else _outputs(made, dq, dk, None, None)


_CACHE_VIEWS = """
    k_cache cache pages kv_heads page_size head_dim
    v_cache cache pages kv_heads page_size head_dim"""
_SCALE_VIEWS = """
    k_scale? f32 pages kv_heads page_size
    v_scale? f32 pages kv_heads page_size"""


def _by_cache_type(plan: _Plan) -> dict:
    return {dtype: plan.typed(cache=dtype)
            for dtype in (torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn)}


_WRITE = _by_cache_type(_Plan("b200_cache_write", """
    k x tokens kv_heads head_dim
    v x tokens kv_heads head_dim
    slots i64 tokens""" + _CACHE_VIEWS + _SCALE_VIEWS + """
    workspace i32 words"""))

_READ = _by_cache_type(_Plan("b200_cache_read", _CACHE_VIEWS + """
    slots i64 tokens""" + _SCALE_VIEWS + """
    k_out= rows tokens kv_heads head_dim
    v_out= rows tokens kv_heads head_dim
    workspace i32 words"""))
_READ = {(store, rows): plan.typed(rows=rows) for store, plan in _READ.items()
         for rows in (torch.float16, torch.bfloat16) if store.itemsize == 1 or store is rows}

_ATTENTION = _by_cache_type(_Plan("b200_paged_attention", """
    q x batch heads head_dim""" + _CACHE_VIEWS + _SCALE_VIEWS + """
    block_table i32 batch columns
    lengths i32 batch
    out= x batch heads head_dim
    lse? f32 batch heads
    partial~ f32 scratch
    workspace i32 words""", "scratch"))


def _cache_type(k_cache, k_scale, v_scale, rows: torch.dtype | None) -> torch.dtype:
    """The type of a cache that goes with its scales and, in 16 bits, with the rows' type."""
    if not isinstance(k_cache, torch.Tensor):
        raise TypeError("k_cache must be a torch.Tensor")
    store = k_cache.dtype
    if store not in _WRITE:
        raise TypeError(f"k_cache must be float16, bfloat16, int8 or float8_e4m3fn, got {store}")
    if store.itemsize == 1:
        if k_scale is None or v_scale is None:
            raise ValueError("an 8-bit cache needs k_scale and v_scale")
    else:
        if k_scale is not None or v_scale is not None:
            raise ValueError("a 16-bit cache has no scales")
        if rows is not None and rows is not store:
            raise TypeError(f"k_cache must have dtype {rows}, torch.int8 or torch.float8_e4m3fn, got {store}")
    return store


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
    rows = _float_type("k", k, (torch.float16, torch.bfloat16))
    store = _cache_type(k_cache, k_scale, v_scale, rows)
    _WRITE[store](device, (k, v, slots, k_cache, v_cache, k_scale, v_scale, _status(device)), (), None,
                  _CODES[rows], _CODES[store])
    return k_cache, v_cache


def cache_read(k_cache, v_cache, slots, k_scale=None, v_scale=None, *, dtype=None, k_out=None, v_out=None):
    """The rows of ``slots`` out of a cache that ``cache_write`` filled, ``(k, v)`` of shape (tokens, heads,
    head_dim): of a 16-bit cache as they are, of an 8-bit one as code * scale in ``dtype`` (f16 or bf16, the
    default).  Negative slots give zeros, and so do slots behind the cache, which ``workspace_status`` reports."""
    device = _cuda_device(k_cache)
    store = _cache_type(k_cache, k_scale, v_scale, None)
    if dtype is None:
        dtype = store if store.itemsize == 2 else torch.bfloat16 if k_out is None else k_out.dtype
    plan = _READ.get((store, dtype))
    if plan is None:
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"dtype must be torch.float16 or torch.bfloat16, got {dtype}")
        raise TypeError(f"a {store} cache gives its rows as they are, not as {dtype}")
    made = plan(device, (k_cache, v_cache, slots, k_scale, v_scale, ... if k_out is None else k_out,
                         ... if v_out is None else v_out, _status(device)), (), None, _CODES[dtype], _CODES[store])
    return made if len(made) == 2 else _outputs(made, k_out, v_out)


def paged_attention(q, k_cache, v_cache, block_table, lengths, scale: float, *, k_scale=None, v_scale=None, out=None,
                    return_lse: bool = False):
    """Attention of one new token a sequence: ``q`` (batch, heads, head_dim) over the first ``lengths[b]`` rows of
    each sequence in a paged cache (``cache_write``), whose pages row ``b`` of ``block_table`` (batch, columns)
    names in order; both int32.  heads is a multiple of the cache's heads, neighbouring query heads share a key
    head; head_dim is 64 or 128.  A sequence of length 0 gets zeros (and lse -infinity).  What lies behind a
    sequence, in its last page or in the table, is never used.  A page outside the cache is left out, a length
    past the table is cut there, and ``workspace_status`` reports both; a sequence that has lost all its positions
    gets NaN.  Infinite values give infinities; infinities and NaN among the values cost a call time.  Returns ``out``, or ``(out, lse)``
    with the natural logarithm of the sums (f32)."""
    device = _cuda_device(q)
    rows = _float_type("q", q, (torch.float16, torch.bfloat16))
    store = _cache_type(k_cache, k_scale, v_scale, rows)
    if q.dim() != 3 or k_cache.dim() != 4 or not isinstance(block_table, torch.Tensor) or block_table.dim() != 2:
        raise ValueError("q is a (batch, heads, head_dim) tensor, k_cache (pages, heads, page_size, head_dim), "
                         "block_table (batch, columns)")
    batch, heads, head_dim = q.shape
    _, kv_heads, page_size, _ = k_cache.shape
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} query heads are not a multiple of the cache's {kv_heads}")
    words = _scratch_size("b200_paged_attention_scratch", device, batch, heads, kv_heads, head_dim,
                          block_table.shape[1] * page_size, _CODES[store])
    made = _ATTENTION[store](device, (q, k_cache, v_cache, k_scale, v_scale, block_table, lengths,
                                      ... if out is None else out, ... if return_lse else None, ..., _status(device)),
                             (words,), float(scale), _CODES[rows], _CODES[store])
    if not return_lse:
        return made[0] if out is None else out
    return made if out is None else (out, made[0])


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
