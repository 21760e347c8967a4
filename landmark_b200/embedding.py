"""Embedding rows and their gradient (``gnr_embedding_lookup``, ``gnr_embedding_grad``).

``embedding`` looks rows of a table up: the appearance latent of every ray or sample of an ``encode_app`` model
(``compute_app_latent``, app/models/gridnerf_sequential.py:429-437, does it with one row for all), or any other table's rows.
``embedding_backward`` is its gradient and, read the other way, the sum of the rows that share an index: samples into rays.
Both are differentiable, each being the other's gradient; forward-mode tangents go through the same operators.

Indices are int32 or int64, of any shape and strides.  A negative one is a masked place: it looks up zeros and adds nothing.
One that is not below the number of rows looks up NaN and adds nothing (only the device sees it, so no error is raised).
Sums are fp32 in an order that only the inputs decide: equal inputs give equal bits.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import check, lib

_TYPES = {torch.float32: _lib.FP32, torch.float16: _lib.FP16, torch.bfloat16: _lib.BF16}
_INDEX_BITS = {torch.int64: 64, torch.int32: 32}


class _Here:
    """Stands for the device guard where the device is the current one."""

    def __enter__(self):
        pass

    def __exit__(self, *exc):
        pass


_here = _Here()


def _on(index: int):
    return _here if index == _current_device() else torch.cuda.device(index)


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# the same without a Stream object and a look at CUDA's initialisation in between (2 us a call), where this torch has them
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _kind(what: str, t: torch.Tensor) -> int:
    kind = _TYPES.get(t.dtype)
    if kind is None:
        raise TypeError(f"{what} must be float32, float16 or bfloat16, got {t.dtype}")
    if not t.is_cuda or t.layout is not torch.strided:
        raise ValueError(f"{what} must be a dense CUDA tensor, got {t.layout} on {t.device}")
    return kind


def _index_bits(indices: torch.Tensor, index: int) -> int:
    bits = _INDEX_BITS.get(indices.dtype)
    if bits is None:
        raise TypeError(f"indices must be int64 or int32, got {indices.dtype}")
    if indices.get_device() != index:
        raise ValueError(f"indices on {indices.device}, values on cuda:{index}")
    return bits


def _rows(t: torch.Tensor):
    """``t [n, d]`` with neighbouring values next to each other and rows that do not overlap, and the rows' distance."""
    if t.is_neg():  # a view with its sign to come, as the imaginary part of a conjugate
        t = t.resolve_neg()
    if t.is_contiguous():
        return t, t.shape[1]
    if t.shape[0] > 1 and (t.stride(1) == 1 or t.shape[1] == 1) and t.stride(0) >= t.shape[1]:
        return t, t.stride(0)
    return t.contiguous(), t.shape[1]


def _lookup(indices: torch.Tensor, weight: torch.Tensor, scale: float) -> torch.Tensor:
    kind, device = _kind("weight", weight), weight.get_device()
    bits = _index_bits(indices, device)
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError(f"weight must be [rows, dim] with a value at least, got {tuple(weight.shape)}")
    rows, dim = weight.shape
    weight, stride = _rows(weight)
    n = indices.numel()
    out = weight.new_empty((*indices.shape, dim))
    if n:
        indices = indices.contiguous()
        with _on(device):
            check(lib.gnr_embedding_lookup(weight.data_ptr(), kind, rows, dim, stride, indices.data_ptr(), bits, n, scale, out.data_ptr(), dim,
                                           _raw_stream(device)), "gnr_embedding_lookup")
    return out


def _rows_share(a: int, a_rows: int, a_stride: int, a_bytes: int, b: int, b_rows: int, b_stride: int, b_bytes: int) -> bool:
    """Whether rows of ``a_bytes`` at a, a + a_stride ... share memory with those at b: columns of one buffer beside each other do not."""
    if a + (a_rows - 1) * a_stride + a_bytes <= b or b + (b_rows - 1) * b_stride + b_bytes <= a:
        return False
    if a_rows > b_rows:  # (the loop goes over the fewer rows)
        a, a_rows, a_stride, a_bytes, b, b_rows, b_stride, b_bytes = b, b_rows, b_stride, b_bytes, a, a_rows, a_stride, a_bytes
    if a_stride == b_stride:  # only the rows' distance counts: one row of a against all that b's may be beside it
        b, b_rows, a_rows = b - (a_rows - 1) * b_stride, a_rows + b_rows - 1, 1
    for row in range(a, a + a_rows * a_stride, a_stride) if a_rows > 1 else (a,):
        first = max(0, (row - b - b_bytes) // b_stride + 1)  # the first row of b that ends behind the beginning of this one
        if first < b_rows and b + first * b_stride < row + a_bytes:
            return True
    return False


_workspace_bytes: dict = {}  # sizes of a call -> bytes the library asks for


def _workspace_need(n: int, rows: int, dim: int) -> int:
    need = _workspace_bytes.get((n, rows, dim))
    if need is None:
        size = C.c_size_t(0)
        check(lib.gnr_embedding_grad_workspace_bytes(n, rows, dim, C.byref(size)), "gnr_embedding_grad_workspace_bytes")
        if len(_workspace_bytes) > 256:
            _workspace_bytes.clear()
        need = _workspace_bytes[n, rows, dim] = size.value
    return need


def _gradient(grad: torch.Tensor, indices: torch.Tensor, scale: float, padding_idx: Optional[int], out: torch.Tensor,
              accumulate: bool, written: bool) -> torch.Tensor:
    kind, device, n = _kind("grad_output", grad), grad.get_device(), indices.numel()
    bits = _index_bits(indices, device)
    rows, dim = out.shape
    grad, stride = _rows(grad if grad.dim() == 2 else grad.reshape(n, dim))
    indices = indices.contiguous()
    if written:  # `out` is the caller's: it must not be what the kernels read
        size = out.element_size()
        at, step, width = out.data_ptr(), (out.stride(0) if rows > 1 else dim) * size, dim * size
        if n and (_rows_share(at, rows, step, width, grad.data_ptr(), n, stride * grad.element_size(), dim * grad.element_size())
                  or _rows_share(at, rows, step, width, indices.data_ptr(), 1, n * bits // 8, n * bits // 8)):
            raise ValueError("out shares memory with grad_output or indices")
    with _on(device):
        need = _workspace_need(n, rows, dim)
        ws = torch.empty(need, dtype=torch.uint8, device=grad.device) if need else None
        check(lib.gnr_embedding_grad(grad.data_ptr(), kind, dim, stride, indices.data_ptr(), bits, n, rows,
                                     -1 if padding_idx is None else padding_idx, scale, accumulate, out.data_ptr(), _TYPES[out.dtype],
                                     out.stride(0) if rows > 1 else dim, ws.data_ptr() if need else None, need, _raw_stream(device)), "gnr_embedding_grad")
    return out


def _no_capture(what: str):
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"the backward pass of {what} cannot be captured into a CUDA graph: torch would add the gradient to the leaf on the "
                           "stream of an earlier pass.  Capture embedding() and embedding_backward() themselves, without autograd")


def _has_tangent(t: torch.Tensor) -> bool:
    """Whether forward-mode differentiation goes through ``t`` (asked only inside a dual level, where this torch says so cheaply)."""
    return getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(t).tangent is not None


def _differentiated(t: torch.Tensor) -> bool:
    return (t.requires_grad and torch.is_grad_enabled()) or _has_tangent(t)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, indices, weight, scale, padding_idx):
        ctx.save_for_backward(indices)
        ctx.save_for_forward(indices)
        ctx.args = weight.shape[0], scale, padding_idx, weight.dtype
        return _lookup(indices, weight, scale)

    @staticmethod
    def backward(ctx, grad):
        _no_capture("embedding")
        rows, scale, padding_idx, dtype = ctx.args
        return None, embedding_backward(grad, ctx.saved_tensors[0], rows, scale=scale, padding_idx=padding_idx, dtype=dtype), None, None

    @staticmethod
    def jvp(ctx, _, tangent, *rest):  # the lookup is linear in the table
        return embedding(ctx.saved_tensors[0], tangent, scale=ctx.args[1], padding_idx=ctx.args[2])


class _EmbeddingBackward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, grad, indices, num_rows, scale, padding_idx, dtype):
        ctx.save_for_backward(indices)
        ctx.save_for_forward(indices)
        ctx.args = scale, padding_idx, grad.dtype, grad.shape
        ctx.result = num_rows, dtype
        return _new_gradient(grad, indices, num_rows, scale, padding_idx, dtype)

    @staticmethod
    def backward(ctx, grad):
        _no_capture("embedding_backward")
        scale, padding_idx, dtype, shape = ctx.args
        indices = ctx.saved_tensors[0]
        indices = torch.where((indices == (-1 if padding_idx is None else padding_idx)) | (indices >= grad.shape[0]), -1, indices)
        return embedding(indices, grad, scale=scale).to(dtype).reshape(shape), None, None, None, None, None

    @staticmethod
    def jvp(ctx, tangent, *rest):  # the sum is linear in what it sums
        num_rows, dtype = ctx.result
        return embedding_backward(tangent, ctx.saved_tensors[0], num_rows, scale=ctx.args[0], padding_idx=ctx.args[1], dtype=dtype)


def _new_gradient(grad, indices, num_rows, scale, padding_idx, dtype):
    return _gradient(grad, indices, scale, padding_idx, grad.new_empty((num_rows, grad.shape[-1]), dtype=dtype), False, False)


def _check_padding(padding_idx: int, rows: int) -> int:
    if not -rows <= padding_idx < rows:
        raise ValueError(f"padding_idx {padding_idx} is not a row of {rows}")
    return padding_idx % rows


def embedding(indices: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[indices]``: rows of ``weight [rows, dim]`` (float32, float16 or bfloat16), shape ``[*indices.shape, dim]``.

    The product is taken in fp32 and rounded once.  ``padding_idx``: a row that gets no gradient."""
    if padding_idx is not None:
        padding_idx = _check_padding(padding_idx, weight.shape[0])
    if _differentiated(weight):
        return _Embedding.apply(indices, weight, float(scale), padding_idx)
    return _lookup(indices, weight, float(scale))


def embedding_backward(grad_output: torch.Tensor, indices: torch.Tensor, num_rows: int, *, scale: float = 1.0, padding_idx: Optional[int] = None,
                       dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """Gradient of ``embedding`` for its weight: row ``v`` of the result is ``scale`` times the sum of the rows
    ``grad_output[t]`` with ``indices[t] == v``, and zeros where there is none; ``grad_output [*indices.shape, dim]``.

    ``dtype``: the result's type (that of ``grad_output``).  ``out [num_rows, dim]``: where it is written, or with
    ``accumulate`` added to; neighbouring values of a row next to each other, no memory shared with ``grad_output`` or ``indices``.  ``padding_idx``: a row
    that gets nothing."""
    _kind("grad_output", grad_output)
    if grad_output.dim() != indices.dim() + 1 or grad_output.shape[:-1] != indices.shape or grad_output.shape[-1] == 0:
        raise ValueError(f"grad_output {tuple(grad_output.shape)} does not fit indices {tuple(indices.shape)}")
    num_rows = int(num_rows)
    if num_rows < 1:
        raise ValueError(f"num_rows must be positive, got {num_rows}")
    if padding_idx is not None:
        padding_idx = _check_padding(padding_idx, num_rows)
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        if dtype is None:
            dtype = grad_output.dtype
        elif dtype not in _TYPES:
            raise TypeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
        if _differentiated(grad_output):
            return _EmbeddingBackward.apply(grad_output, indices, num_rows, float(scale), padding_idx, dtype)
        return _new_gradient(grad_output, indices, num_rows, float(scale), padding_idx, dtype)
    _kind("out", out)
    if dtype is not None and dtype != out.dtype:
        raise TypeError(f"out is {out.dtype}, dtype {dtype}")
    if tuple(out.shape) != (num_rows, grad_output.shape[-1]) or out.device != grad_output.device:
        raise ValueError(f"out {tuple(out.shape)} on {out.device} must be {(num_rows, grad_output.shape[-1])} on {grad_output.device}")
    if out.is_neg() or (out.stride(1) != 1 and out.shape[1] > 1) or (num_rows > 1 and out.stride(0) < out.shape[1]):
        raise ValueError(f"out must have neighbouring values next to each other and rows that do not overlap, got strides {out.stride()}")
    if _differentiated(grad_output) or _differentiated(out):
        raise RuntimeError("embedding_backward writes out in place and is not differentiable then")
    _gradient(grad_output, indices, float(scale), padding_idx, out, bool(accumulate), True)
    increment_version(out)  # a backward pass over what was computed from the old values is an error
    return out
