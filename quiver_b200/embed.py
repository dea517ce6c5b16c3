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

__all__ = ["ACTIVATIONS", "Adapter", "embedding_grad", "embedding_lookup", "linear", "linear_grad"]

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ID_TYPES = {torch.int32: 0, torch.int64: 1}
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def _dtype_code(t: torch.Tensor, what: str) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise ValueError(f"{what}: expected float32, float16 or bfloat16, got {t.dtype}") from None


def _activation_code(activation: str) -> int:
    try:
        return ACTIVATIONS[activation]
    except KeyError:
        raise ValueError(f"unknown activation '{activation}' (expected one of "
                         f"{', '.join(ACTIVATIONS)})") from None


def _cuda(t, what: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what}: expected a CUDA tensor")
    return t


def _like(t, ref: torch.Tensor, what: str, shape) -> torch.Tensor:
    _cuda(t, what)
    if t.dtype != ref.dtype:
        raise ValueError(f"{what}: expected {ref.dtype}, got {t.dtype}")
    if t.device != ref.device:
        raise ValueError(f"{what}: expected a tensor on {ref.device}, got {t.device}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    return t


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A 2-D tensor whose rows are contiguous and do not overlap, copied only when t's are not."""
    if (t.stride(1) == 1 or t.shape[1] == 1) and (t.stride(0) >= t.shape[1] or t.shape[0] <= 1):
        return t
    return t.contiguous()


def _ids(ids: torch.Tensor, device) -> Tuple[torch.Tensor, int]:
    _cuda(ids, "ids")
    if ids.dtype not in _ID_TYPES:
        raise ValueError(f"ids: expected int32 or int64, got {ids.dtype}")
    if ids.device != device:
        raise ValueError(f"ids: expected a tensor on {device}, got {ids.device}")
    return ids.contiguous(), _ID_TYPES[ids.dtype]


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _workspace(nbytes: int, device):
    if nbytes == 0:
        return None, 0
    return torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes


def _check_out(out, shape, dtype, device):
    """A caller's result tensor: rows contiguous, or a new tensor when None."""
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    _cuda(out, "out")
    if out.dtype != dtype or out.device != device or tuple(out.shape) != tuple(shape):
        raise ValueError(f"out: expected {dtype} {tuple(shape)} on {device}")
    if out.requires_grad:
        raise ValueError("out: must not require a gradient")
    if not out.is_contiguous():
        raise ValueError("out: expected a contiguous tensor")
    return out


# ---- embedding tables -------------------------------------------------------------------------------


def _lookup(table, ids, scale, out):
    if table.dim() != 2:
        raise ValueError(f"table: expected [rows, dim], got shape {tuple(table.shape)}")
    code = _dtype_code(table, "table")
    i, id_code = _ids(ids, table.device)
    t = _rows(table)
    rows, dim = t.shape
    out = _check_out(out, tuple(ids.shape) + (dim,), table.dtype, table.device)
    check(lib().qv_embedding_lookup_device(table.device.index, code, t.data_ptr(), rows, dim,
                                           max(t.stride(0), dim), id_code, i.data_ptr(), i.numel(),
                                           scale, out.data_ptr(), dim, _stream(table.device)))
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
    _cuda(table, "table")
    if out is None and torch.is_grad_enabled() and table.requires_grad:
        return _Lookup.apply(table, ids, float(scale))
    return _lookup(table, ids, float(scale), out)


def embedding_grad(grad: torch.Tensor, ids: torch.Tensor, rows: int, scale: float = 1.0, *,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The table's gradient of :func:`embedding_lookup`: ``[rows, dim]`` with
    ``scale * sum of grad[i] over ids[i] == r`` in row r, zeros where no id points. ``grad`` is
    ``[*ids.shape, dim]``; ids outside ``[0, rows)`` take no gradient. Sums are float32 in the order
    of the ids, so equal calls give equal bits."""
    _cuda(grad, "grad")
    code = _dtype_code(grad, "grad")
    i, id_code = _ids(ids, grad.device)
    if grad.dim() < 1 or tuple(grad.shape[:-1]) != tuple(ids.shape):
        raise ValueError(f"grad: expected shape {tuple(ids.shape)} + (dim,), got "
                         f"{tuple(grad.shape)}")
    rows = int(rows)
    if rows < 0:
        raise ValueError("rows must not be negative")
    dim = grad.shape[-1]
    g = _rows(grad.reshape(-1, dim) if grad.dim() != 2 else grad)
    out = _check_out(out, (rows, dim), grad.dtype, grad.device)
    n = i.numel()
    size = C.c_size_t()
    check(lib().qv_embedding_grad_workspace(n, rows, dim, C.byref(size)))
    ws, nbytes = _workspace(size.value, grad.device)
    check(lib().qv_embedding_grad_device(grad.device.index, code, g.data_ptr(),
                                         max(g.stride(0), dim), id_code, i.data_ptr(), n, rows,
                                         dim, float(scale), out.data_ptr(), dim,
                                         ws.data_ptr() if ws is not None else None, nbytes,
                                         _stream(grad.device)))
    return out


# ---- linear adapters -----------------------------------------------------------------------------


def _linear(x, weight, bias, residual, activation, out_dtype, want_preact, out=None):
    """The checked call: (out, preact or None), both shaped [*x.shape[:-1], n]."""
    _cuda(x, "x")
    code = _dtype_code(x, "x")
    act = _activation_code(activation)
    _cuda(weight, "weight")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"expected x [..., k] and weight [n, k], got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    n, k = weight.shape
    shape = tuple(x.shape[:-1]) + (n,)
    _like(weight, x, "weight", (n, k))
    if bias is not None:
        bias = _like(bias, x, "bias", (n,)).contiguous()
    if out_dtype is None:
        out_dtype = x.dtype
    if out_dtype not in (x.dtype, torch.float32):
        raise ValueError(f"out_dtype: expected {x.dtype} or torch.float32, got {out_dtype}")
    out = _check_out(out, shape, out_dtype, x.device)
    x2 = _rows(x.reshape(-1, k) if x.dim() != 2 else x)
    w = _rows(weight)
    m = x2.shape[0]
    a = _native.qv_linear(code, _DTYPES[out_dtype], act, m, n, k, x2.data_ptr(),
                          max(x2.stride(0), k), w.data_ptr(), max(w.stride(0), k),
                          bias.data_ptr() if bias is not None else None)
    if residual is not None:
        r = _like(residual, x, "residual", shape)
        r = r.reshape(-1, n) if r.dim() != 2 else r
        if not (r.shape[0] > 1 and r.stride(0) == 0 and (r.stride(1) == 1 or n == 1)):
            r = _rows(r)
        a.residual, a.residual_stride = r.data_ptr(), r.stride(0) if m > 1 else n
    preact = None
    if want_preact:
        preact = torch.empty(shape, dtype=x.dtype, device=x.device)
        a.preact, a.preact_stride = preact.data_ptr(), n
    a.out, a.out_stride = out.data_ptr(), n
    size = C.c_size_t()
    device = x.device.index
    check(lib().qv_linear_workspace(device, C.byref(a), C.byref(size)))
    ws, nbytes = _workspace(size.value, x.device)
    check(lib().qv_linear_device(device, C.byref(a), ws.data_ptr() if ws is not None else None,
                                 nbytes, _stream(x.device)))
    return out, preact


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, out_dtype):
        y, preact = _linear(x, weight, bias, residual, activation, out_dtype,
                            activation != "none")
        ctx.save_for_backward(x, weight, preact)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, preact = ctx.saved_tensors
        need = ctx.needs_input_grad
        g = grad.to(x.dtype)  # of a float32 result
        dx, dw, db = (None, None, None)
        if need[0] or need[1] or need[2]:
            dx, dw, db = linear_grad(g, x, weight, preact, ctx.activation, need=need[:3])
        return dx, dw, db, g if need[3] else None, None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
           residual: Optional[torch.Tensor] = None, activation: str = "none",
           out_dtype: Optional[torch.dtype] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``activation(x @ weight.T + bias) + residual`` for x [..., k], weight [n, k], bias [n] and a
    residual of the result's shape [..., n] (an expanded one is not copied). ``activation`` is one of
    :data:`ACTIVATIONS`; ``out_dtype`` may be torch.float32 to leave the result unrounded.
    Differentiable in all four tensors (unless ``out`` is given)."""
    if out is None and torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (x, weight, bias, residual)):
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
    """The gradients (dx, dweight, dbias) of :func:`linear` for ``grad`` = d loss / d result, in x's
    type; those not asked for in ``need`` are None. ``preact`` (from :func:`linear_preact`) may be
    None without an activation. The residual's gradient is ``grad`` itself."""
    _cuda(x, "x")
    code = _dtype_code(x, "x")
    act = _activation_code(activation)
    _cuda(weight, "weight")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"expected x [..., k] and weight [n, k], got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    n, k = weight.shape
    _like(weight, x, "weight", (n, k))
    shape = tuple(x.shape[:-1]) + (n,)
    _like(grad, x, "grad", shape)
    g = _rows(grad.reshape(-1, n) if grad.dim() != 2 else grad)
    x2 = _rows(x.reshape(-1, k) if x.dim() != 2 else x)
    w = _rows(weight)
    m = x2.shape[0]
    a = _native.qv_linear_grad(code, act, m, n, k, g.data_ptr(), max(g.stride(0), n),
                               x2.data_ptr(), max(x2.stride(0), k), w.data_ptr(),
                               max(w.stride(0), k))
    if act != 0:
        if preact is None:
            raise ValueError("preact: needed for the gradient of an activation")
        p = _like(preact, x, "preact", shape)
        p = _rows(p.reshape(-1, n) if p.dim() != 2 else p)
        a.preact, a.preact_stride = p.data_ptr(), max(p.stride(0), n)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
    dw = torch.empty((n, k), dtype=x.dtype, device=x.device) if need[1] else None
    db = torch.empty((n,), dtype=x.dtype, device=x.device) if need[2] else None
    if dx is not None:
        a.dx, a.dx_stride = dx.data_ptr(), k
    if dw is not None:
        a.dweight, a.dweight_stride = dw.data_ptr(), k
    if db is not None:
        a.dbias = db.data_ptr()
    size = C.c_size_t()
    device = x.device.index
    check(lib().qv_linear_grad_workspace(device, C.byref(a), C.byref(size)))
    ws, nbytes = _workspace(size.value, x.device)
    check(lib().qv_linear_grad_device(device, C.byref(a),
                                      ws.data_ptr() if ws is not None else None, nbytes,
                                      _stream(x.device)))
    return dx, dw, db


class Adapter:
    """One linear map for the vectors of an index: ``activation(v W^T + bias)``, plus v itself with
    ``residual=True`` (W square). ``adapter(v)`` gives float32 vectors, ready for
    :meth:`FlatIndex.add_device` and the device searches, which also take it as ``adapter=``."""

    def __init__(self, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                 activation: str = "none", residual: bool = False):
        _cuda(weight, "weight")
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
            return linear(x, self.weight, self.bias, residual=x if self.residual else None,
                          activation=self.activation, out_dtype=torch.float32)

    @property
    def in_dim(self) -> int:
        return self.weight.shape[1]

    @property
    def out_dim(self) -> int:
        return self.weight.shape[0]

    def __repr__(self) -> str:
        return (f"Adapter({self.in_dim} -> {self.out_dim}, activation={self.activation!r}, "
                f"residual={self.residual})")
