"""Embedding tables and linear adapters on the GPU: the trainable front of an index.

An index searches vectors that a model learned. This module holds the two operators between such a
model and the index, with their gradients, on CUDA tensors:

* :func:`embedding_lookup` gathers rows of a table by id with a scale (a search result's unfilled
  ``-1`` slots give rows of zeros); its gradient :func:`embedding_grad` sums by sorted id.
* :func:`linear` computes ``activation(x W^T + bias) + residual`` in one tensor-core kernel; its
  gradients are :func:`linear_grad`. :class:`Adapter` keeps the weights of one such map for the
  device add and search paths (``adapter=``).

``embedding_lookup`` and ``linear`` are differentiable (``torch.autograd``). Inputs are float32,
float16 or bfloat16 tensors of one type and device; sums are float32 in a fixed order and rounded
once. Work goes to PyTorch's current stream of the inputs' device, without host synchronization;
temporaries come from PyTorch's caching allocator on that stream, so calls can be captured into
CUDA graphs. To capture a backward pass, call :func:`embedding_grad` and :func:`linear_grad`
directly, or follow PyTorch's rules for capturing autograd.

    >>> table = torch.randn(32000, 768, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    >>> x = embedding_lookup(table, token_ids, scale=768 ** 0.5)
    >>> y = linear(x, weight, bias, residual=x, activation="gelu")
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _native
from ._native import check, lib

__all__ = ["ACTIVATIONS", "Adapter", "embedding_grad", "embedding_lookup", "linear", "linear_grad",
           "linear_preact"]

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ID_TYPES = {torch.int32: 0, torch.int64: 1}
_GRAD_F32 = 0x100  # QV_GRAD_F32
_RESIDUAL_F32 = 0x100  # QV_RESIDUAL_F32
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


# The handle of PyTorch's current stream, as torch.cuda.current_stream(i).cuda_stream, without
# building a Stream object: that costs as much host time as a kernel launch.
_raw_stream = torch._C._cuda_getCurrentRawStream


def _bad(what: str, expected: str, got) -> ValueError:
    return ValueError(f"{what}: expected {expected}, got {got}")


def _dtype_code(t, what: str) -> int:
    """The element type's code of a CUDA tensor; refuses anything else."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what}: expected a CUDA tensor")
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise _bad(what, "float32, float16 or bfloat16", t.dtype)
    return code


def _activation_code(activation: str) -> int:
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"unknown activation '{activation}' (expected one of "
                         f"{', '.join(ACTIVATIONS)})")
    return code


def _like(t, ref: torch.Tensor, what: str, shape) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != ref.dtype or t.device != ref.device or \
            t.shape != shape:
        if not isinstance(t, torch.Tensor):
            raise _bad(what, "a CUDA tensor", type(t).__name__)
        raise _bad(what, f"{ref.dtype} {tuple(shape)} on {ref.device}",
                   f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A 2-D tensor whose rows are contiguous and do not overlap, copied only when t's are not."""
    rows, cols = t.shape
    s0, s1 = t.stride()
    if (s1 == 1 or cols == 1) and (s0 >= cols or rows <= 1):
        return t
    return t.contiguous()


def _ids(ids, device) -> Tuple[torch.Tensor, int]:
    if not isinstance(ids, torch.Tensor) or not ids.is_cuda:
        raise ValueError("ids: expected a CUDA tensor")
    code = _ID_TYPES.get(ids.dtype)
    if code is None:
        raise _bad("ids", "int32 or int64", ids.dtype)
    if ids.device != device:
        raise _bad("ids", f"a tensor on {device}", ids.device)
    return ids.contiguous(), code


def _check_out(out, shape, dtype, device):
    """A caller's result tensor."""
    if not isinstance(out, torch.Tensor) or out.dtype != dtype or out.device != device or \
            tuple(out.shape) != tuple(shape):
        raise ValueError(f"out: expected {dtype} {tuple(shape)} on {device}")
    if out.requires_grad:
        raise ValueError("out: must not require a gradient")
    if not out.is_contiguous():
        raise ValueError("out: expected a contiguous tensor")
    return out


def _extent(t: torch.Tensor):
    """First and last-past byte address a tensor reaches."""
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * st for n, st in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _apart(out: torch.Tensor, **inputs) -> None:
    """Refuses a caller's result that shares memory with an input."""
    a, b = _extent(out)
    for what, t in inputs.items():
        if t is not None:
            c, d = _extent(t)
            if a < d and c < b:
                raise ValueError(f"out: must not share memory with {what}")


# ---- embedding tables -------------------------------------------------------------------------------


def _lookup(table, ids, scale, out):
    code = _dtype_code(table, "table")
    if table.dim() != 2:
        raise _bad("table", "[rows, dim]", f"shape {tuple(table.shape)}")
    device = table.device
    i, id_code = _ids(ids, device)
    t = _rows(table)
    rows, dim = t.shape
    shape = (*ids.shape, dim)
    if out is None:
        out = table.new_empty(shape)
    else:
        _apart(_check_out(out, shape, table.dtype, device), table=table, ids=ids)
    index = device.index
    check(lib().qv_embedding_lookup_device(index, code, t.data_ptr(), rows, dim,
                                           max(t.stride(0), dim), id_code, i.data_ptr(), i.numel(),
                                           scale, out.data_ptr(), dim, _raw_stream(index)))
    return out


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale = table.shape[0], scale
        return _lookup(table, ids, scale, None)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        return embedding_grad(grad, ids, ctx.rows, ctx.scale), None, None


def embedding_lookup(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, *,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``scale * table[ids]`` for a table [rows, dim] and int32 / int64 ids of any shape: returns
    ``[*ids.shape, dim]``. A negative id (an unfilled search result slot) gives zeros, an id of
    ``rows`` or more a row of NaN. Differentiable in the table (unless ``out`` is given)."""
    if out is None and torch.is_grad_enabled() and getattr(table, "requires_grad", False):
        return _Lookup.apply(table, ids, float(scale))
    return _lookup(table, ids, float(scale), out)


def embedding_grad(grad: torch.Tensor, ids: torch.Tensor, rows: int, scale: float = 1.0, *,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The table's gradient of :func:`embedding_lookup`: ``[rows, dim]`` with
    ``scale * sum of grad[i] over ids[i] == r`` in row r, zeros where no id points. ``grad`` is
    ``[*ids.shape, dim]``; ids outside ``[0, rows)`` take no gradient. Sums are float32 in the order
    of the ids, so equal calls give equal bits."""
    code = _dtype_code(grad, "grad")
    device = grad.device
    i, id_code = _ids(ids, device)
    if grad.dim() < 1 or grad.shape[:-1] != ids.shape:
        raise _bad("grad", f"shape {tuple(ids.shape)} + (dim,)", tuple(grad.shape))
    rows = int(rows)
    if rows < 0:
        raise ValueError("rows must not be negative")
    dim = grad.shape[-1]
    n = i.numel()
    g = _rows(grad if grad.dim() == 2 else grad.reshape(n, dim))
    size = C.c_size_t()
    call = lib()
    check(call.qv_embedding_grad_workspace(n, rows, dim, C.byref(size)))
    if out is None:
        out = grad.new_empty((rows, dim))
    else:
        _apart(_check_out(out, (rows, dim), grad.dtype, device), grad=grad, ids=ids)
    ws = torch.empty(size.value, dtype=torch.uint8, device=device)
    index = device.index
    check(call.qv_embedding_grad_device(index, code, g.data_ptr(), max(g.stride(0), dim), id_code,
                                        i.data_ptr(), n, rows, dim, float(scale), out.data_ptr(),
                                        dim, ws.data_ptr(), size.value, _raw_stream(index)))
    return out


# ---- linear adapters -----------------------------------------------------------------------------


def _linear(x, weight, bias, residual, activation, out_dtype, want_preact, out=None):
    """The checked call: (out, preact or None), both shaped [*x.shape[:-1], n]."""
    code = _dtype_code(x, "x")
    act = _activation_code(activation)
    _dtype_code(weight, "weight")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"expected x [..., k] and weight [n, k], got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    n, k = weight.shape
    _like(weight, x, "weight", (n, k))
    device = x.device
    x2 = _rows(x if x.dim() == 2 else x.reshape(x.numel() // k if k else 0, k))
    m = x2.shape[0]
    shape = (*x.shape[:-1], n)
    w = _rows(weight)
    bias_ptr = residual_ptr = preact = None
    residual_stride = 0
    if bias is not None:
        bias = _like(bias, x, "bias", (n,)).contiguous()  # held until the call is enqueued
        bias_ptr = bias.data_ptr()
    if out_dtype is None:
        out_dtype = x.dtype
    elif out_dtype != x.dtype and out_dtype != torch.float32:
        raise _bad("out_dtype", f"{x.dtype} or torch.float32", out_dtype)
    out_code = _DTYPES[out_dtype]
    if residual is not None:
        r = residual
        if out_code == 0 and code != 0 and getattr(r, "dtype", None) == torch.float32:
            out_code |= _RESIDUAL_F32
            if r.device != device or r.shape != shape:
                raise _bad("residual", f"{tuple(shape)} on {device}", f"{tuple(r.shape)} on {r.device}")
        else:
            _like(r, x, "residual", shape)
        r = r if r.dim() == 2 else r.reshape(m, n)
        if not (r.stride(0) == 0 and (r.stride(1) == 1 or n == 1)):
            r = _rows(r)
        residual_ptr, residual_stride = r.data_ptr(), r.stride(0) if m > 1 else n
    if out is None:
        out = torch.empty(shape, dtype=out_dtype, device=device)
    else:
        _apart(_check_out(out, shape, out_dtype, device), x=x, weight=weight, bias=bias,
               residual=residual)
    if want_preact:
        preact = x.new_empty(shape)
    a = _native.qv_linear(code, out_code, act, m, n, k, x2.data_ptr(),
                          max(x2.stride(0), k), w.data_ptr(), max(w.stride(0), k), bias_ptr,
                          residual_ptr, residual_stride, out.data_ptr(), n,
                          preact.data_ptr() if want_preact else None, n)
    size = C.c_size_t()
    index = device.index
    call, ref = lib(), C.byref(a)
    check(call.qv_linear_workspace(index, ref, C.byref(size)))
    if size.value:
        ws = torch.empty(size.value, dtype=torch.uint8, device=device)
        check(call.qv_linear_device(index, ref, ws.data_ptr(), size.value, _raw_stream(index)))
    else:
        check(call.qv_linear_device(index, ref, None, 0, _raw_stream(index)))
    return out, preact


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, out_dtype):
        y, preact = _linear(x, weight, bias, residual, activation, out_dtype,
                            activation != "none")
        ctx.save_for_backward(x, weight, preact)
        ctx.activation = activation
        ctx.residual_dtype = None if residual is None else residual.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, preact = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = (None, None, None)
        if need[0] or need[1] or need[2]:  # what the forward pass checked
            dx, dw, db = _linear_grad(grad, x, weight, preact, ACTIVATIONS[ctx.activation], need)
        return dx, dw, db, grad.to(ctx.residual_dtype) if need[3] else None, None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
           residual: Optional[torch.Tensor] = None, activation: str = "none",
           out_dtype: Optional[torch.dtype] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``activation(x @ weight.T + bias) + residual`` for x [..., k], weight [n, k], bias [n] and a
    residual of the result's shape [..., n] (an expanded one is not copied). ``activation`` is one of
    :data:`ACTIVATIONS`; ``out_dtype`` may be torch.float32 to leave the result unrounded (the residual
    may then be float32 too). float32 products are off by at most 2^-21 of sum |x||w| beside a float32
    sum's own roundings; float32 results of 16-bit inputs, whose sums the tensor core cuts, by up to
    3.4e-6 of it. Differentiable in all four tensors (unless ``out`` is given)."""
    if out is None and torch.is_grad_enabled() and any(
            [isinstance(t, torch.Tensor) and t.requires_grad for t in (x, weight, bias, residual)]):
        return _Linear.apply(x, weight, bias, residual, activation, out_dtype)
    return _linear(x, weight, bias, residual, activation, out_dtype, False, out)[0]


def linear_preact(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                  residual: Optional[torch.Tensor] = None, activation: str = "none",
                  out_dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`linear` together with the values ahead of the activation, which
    :func:`linear_grad` takes; no autograd."""
    return _linear(x, weight, bias, residual, activation, out_dtype, True)


def linear_grad(grad: torch.Tensor, x: torch.Tensor, weight: torch.Tensor,
                preact: Optional[torch.Tensor] = None, activation: str = "none", *,
                need: Tuple[bool, bool, bool] = (True, True, True)):
    """The gradients (dx, dweight, dbias) of :func:`linear` for ``grad`` = d loss / d result (in x's
    type or float32), in x's type; those not asked for in ``need`` are None. ``preact`` (from
    :func:`linear_preact`) may be None without an activation. The residual's gradient is ``grad``
    itself."""
    _dtype_code(x, "x")
    act = _activation_code(activation)
    _dtype_code(weight, "weight")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"expected x [..., k] and weight [n, k], got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    n, k = weight.shape
    _like(weight, x, "weight", (n, k))
    shape = (*x.shape[:-1], n)
    if getattr(grad, "dtype", None) == torch.float32:
        if grad.device != x.device or grad.shape != shape:
            raise _bad("grad", f"{tuple(shape)} on {x.device}", f"{tuple(grad.shape)} on {grad.device}")
    else:
        _like(grad, x, "grad", shape)
    if act != 0:
        if preact is None:
            raise ValueError("preact: needed for the gradient of an activation")
        _like(preact, x, "preact", shape)
    return _linear_grad(grad, x, weight, preact, act, need)


def _linear_grad(grad, x, weight, preact, act, need):
    """:func:`linear_grad` of checked arguments."""
    n, k = weight.shape
    x2 = _rows(x if x.dim() == 2 else x.reshape(x.numel() // k if k else 0, k))
    m = x2.shape[0]
    g = _rows(grad if grad.dim() == 2 else grad.reshape(m, n))
    w = _rows(weight)
    preact_ptr, preact_stride = None, 0
    if act != 0:
        p = _rows(preact if preact.dim() == 2 else preact.reshape(m, n))
        preact_ptr, preact_stride = p.data_ptr(), max(p.stride(0), n)
    dx = x.new_empty(x.shape) if need[0] else None
    dw = x.new_empty((n, k)) if need[1] else None
    db = x.new_empty((n,)) if need[2] else None
    code = _DTYPES[x.dtype]
    if code and grad.dtype == torch.float32:
        code |= _GRAD_F32
    a = _native.qv_linear_grad(code, act, m, n, k, g.data_ptr(), max(g.stride(0), n),
                               x2.data_ptr(), max(x2.stride(0), k), w.data_ptr(),
                               max(w.stride(0), k), preact_ptr, preact_stride,
                               dx.data_ptr() if need[0] else None, k,
                               dw.data_ptr() if need[1] else None, k,
                               db.data_ptr() if need[2] else None)
    size = C.c_size_t()
    index = x.device.index
    call, ref = lib(), C.byref(a)
    check(call.qv_linear_grad_workspace(index, ref, C.byref(size)))
    ws = torch.empty(size.value, dtype=torch.uint8, device=x.device)
    check(call.qv_linear_grad_device(index, ref, ws.data_ptr(), size.value, _raw_stream(index)))
    return dx, dw, db


class Adapter:
    """One linear map for the vectors of an index: ``activation(v W^T + bias)``, plus v itself with
    ``residual=True`` (W square). The product takes v in the weight's type; what is added is v as it
    is. ``adapter(v)`` gives float32 vectors, ready for
    :meth:`FlatIndex.add_device` and the device searches, which also take it as ``adapter=``. The same
    vector in another batch may differ in its last bits (sums run in another order by the batch's
    size, float32 ones on other parts where the batch holds rows of wide range)."""

    def __init__(self, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                 activation: str = "none", residual: bool = False):
        _dtype_code(weight, "weight")
        _activation_code(activation)
        if weight.dim() != 2:
            raise ValueError(f"weight: expected [n, k], got shape {tuple(weight.shape)}")
        if bias is not None:
            _like(bias, weight, "bias", (weight.shape[0],))
        if residual and weight.shape[0] != weight.shape[1]:
            raise ValueError("a residual adapter needs a square weight")
        self.weight, self.bias = weight, bias
        self.activation, self.residual = activation, bool(residual)

    def __call__(self, vectors: torch.Tensor) -> torch.Tensor:
        with torch.no_grad():
            x = vectors.to(self.weight.dtype)
            skip = None
            if self.residual:
                skip = x if vectors.dtype == x.dtype else vectors.to(torch.float32)
            return linear(x, self.weight, self.bias, residual=skip, activation=self.activation,
                          out_dtype=torch.float32)

    @property
    def in_dim(self) -> int:
        return self.weight.shape[1]

    @property
    def out_dim(self) -> int:
        return self.weight.shape[0]

    def __repr__(self) -> str:
        return (f"Adapter({self.in_dim} -> {self.out_dim}, activation={self.activation!r}, "
                f"residual={self.residual})")
