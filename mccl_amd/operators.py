"""Operators of a data-parallel training step around the gradients that the reduce queue
carries: layer norm, dropout, both in one pass over the seam of a transformer block, and the
loss at the end of a language model.

Each comes three ways: `*_forward` / `*_backward` on tensors, a differentiable function of
the same name without a suffix, and for training code `MaskStream`, which hands out the
masks of dropout.  Every arithmetic launch is a hand-written HIP kernel inside libmcclx.so.

The kernels run on torch's current stream, not on the reduce queue: they are the producers
whose gradients a bucket's allreduce waits for.  A queue (`hip_kernels_init`) must exist: it
names the device and counts the launches.  Scratch memory comes from torch's allocator for
each call.  A call may be recorded into a graph, which keeps its arguments: the seed and offset of a dropout too, so that
every replay draws the mask of the recording.  A training step that is replayed keeps its dropouts outside the graph, or p at 0.

Tensors are matrices of rows: the last dimension is the row.  Rows may lie further apart than
they are long (a slice of a wider tensor is read in place); any other layout is copied first.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _lib as L
from ._lib import MCCLError
from .harness import _reader
from .kernels import _DTYPE, _q, dtype_code

__all__ = ["layer_norm", "layer_norm_forward", "layer_norm_backward", "dropout", "dropout_forward", "dropout_backward",
           "dropout_add_layer_norm", "dropout_add_layer_norm_forward", "dropout_add_layer_norm_backward", "MaskStream",
           "linear_cross_entropy", "linear_cross_entropy_forward", "linear_cross_entropy_backward"]

_M64 = (1 << 64) - 1


def _stream(q) -> int:
    return torch._C._cuda_getCurrentRawStream(q.device)   # (current_stream() makes an object of it, 1 us)


def _on_gpu(q, t: torch.Tensor, what: str) -> None:
    if t.get_device() != q.device:     # (-1 on the CPU)
        if not t.is_cuda:
            raise MCCLError(f"[MCCL] {what}: tensor must live on the GPU; got {t.device.type} tensor")
        raise MCCLError(f"[MCCL] {what}: tensor lives on GPU {t.device.index}, the queue on {q.device}")


def _rows(q, t: torch.Tensor, what: str) -> Tuple[torch.Tensor, int, int, int]:
    """(tensor, rows, cols, elements from a row to the next)."""
    _on_gpu(q, t, what)
    if t.dim() == 0:
        raise MCCLError(f"[MCCL] {what}: a scalar has no rows")
    cols = t.shape[-1]
    if t.is_contiguous():
        return t, t.numel() // cols if cols else 0, cols, cols
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= cols:
        return t, t.shape[0], cols, t.stride(0)
    if t.stride(-1) == 1 and t.numel():
        try:
            flat = t.view(-1, cols)
        except RuntimeError:
            flat = t
        if flat.dim() == 2 and flat.stride(0) >= cols:
            return flat, flat.shape[0], cols, flat.stride(0)
    t = t.contiguous()
    return t, t.numel() // cols if cols else 0, cols, cols


def _same(a: torch.Tensor, b: torch.Tensor, what: str) -> None:
    if a.shape != b.shape:
        raise MCCLError(f"[MCCL] {what}: shape {tuple(b.shape)} beside {tuple(a.shape)}")
    if a.dtype != b.dtype:
        raise MCCLError(f"[MCCL] {what}: dtype {b.dtype} beside {a.dtype}")


def _params(q, x: torch.Tensor, cols: int, *named) -> int:
    """Checks weight and bias (None: left out) and returns their dtype's code."""
    code = None
    for t, what in named:
        if t is None:
            continue
        _on_gpu(q, t, what)
        if t.dim() != 1 or t.shape[0] != cols or not t.is_contiguous():
            raise MCCLError(f"[MCCL] {what}: expected {cols} adjacent elements, got shape {tuple(t.shape)}")
        if t.dtype not in (x.dtype, torch.float32):
            raise MCCLError(f"[MCCL] {what}: dtype {t.dtype} beside {x.dtype}", L.ERR_UNSUPPORTED)
        if code is None:
            code = t.dtype
        elif t.dtype != code:
            raise MCCLError(f"[MCCL] {what}: weight and bias differ in dtype")
    return dtype_code(x) if code is None else _DTYPE[code]


def _like(x: torch.Tensor) -> torch.Tensor:
    """A new tensor of x's shape, its rows adjacent."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _stats(q, t: torch.Tensor, rows: int, what: str) -> torch.Tensor:
    _on_gpu(q, t, what)
    if t.dtype != torch.float32 or t.numel() != rows or not t.is_contiguous():
        raise MCCLError(f"[MCCL] {what}: expected {rows} adjacent float32 values, got {t.dtype} of shape {tuple(t.shape)}")
    return t


def _mask(p: float, seed: int, offset: int) -> Tuple[float, int, int]:
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise MCCLError(f"[MCCL] dropout: p={p} outside 0..1")
    return p, int(seed) & _M64, int(offset) & _M64


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# ---- layer norm, with or without the seam ----------------------------------------

def _norm_forward(q, x, residual, weight, bias, p, seed, offset, eps, keep_sum):
    native = _reader()
    if native is not None:
        done = native._norm_forward(q.handle.value, q.device, x, residual, weight, bias, p, seed, offset, eps, keep_sum)
        if done is not None:
            L.check(done[0])
            return done[1:]
    xr, rows, cols, x_stride = _rows(q, x, "x")
    r_stride = 0
    if residual is not None:
        _same(x, residual, "residual")
        residual, _, _, r_stride = _rows(q, residual, "residual")
    param = _params(q, x, cols, (weight, "weight"), (bias, "bias"))
    y = _like(x)
    s = torch.empty_like(y) if keep_sum else None
    mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
    rstd = torch.empty_like(mean)
    a = L.Norm(dtype_code(x), param, rows, cols, float(eps), p, seed, offset, _ptr(weight), _ptr(bias), mean.data_ptr(),
               rstd.data_ptr(), xr.data_ptr(), _ptr(residual), y.data_ptr(), _ptr(s))
    a.x_stride = x_stride
    a.residual_stride = r_stride
    L.check(L.lib().mcclx_layer_norm_forward(q.handle, _stream(q), C.byref(a)))
    return y, s, mean, rstd


def _norm_backward(q, dy, ds, s, mean, rstd, weight, p, seed, offset, with_x, with_residual, with_weight, bias_dtype):
    """bias_dtype: dbias's, None: no dbias."""
    native = _reader()
    if native is not None:
        done = native._norm_backward(q.handle.value, q.device, dy, ds, s, mean, rstd, weight, p, seed, offset, with_x, with_residual,
                                     with_weight, -1 if bias_dtype is None else _DTYPE.get(bias_dtype, -2))
        if done is not None:
            L.check(done[0])
            return done[1:]
    _same(s, dy, "dy")
    sr, rows, cols, s_stride = _rows(q, s, "s")
    dyr, _, _, dy_stride = _rows(q, dy, "dy")
    ds_stride = 0
    if ds is not None:
        _same(s, ds, "ds")
        ds, _, _, ds_stride = _rows(q, ds, "ds")
    param = _params(q, s, cols, (weight, "weight"))
    if bias_dtype is not None:
        if bias_dtype not in ((s.dtype, torch.float32) if weight is None else (weight.dtype,)):
            raise MCCLError(f"[MCCL] bias: dtype {bias_dtype} beside {s.dtype if weight is None else weight.dtype}", L.ERR_UNSUPPORTED)
        param = _DTYPE[bias_dtype]
    _stats(q, mean, rows, "mean")
    _stats(q, rstd, rows, "rstd")
    lib = L.lib()
    dx = _like(s) if with_x else None
    dresidual = _like(s) if with_residual else None
    dweight = torch.empty_like(weight) if with_weight and weight is not None else None
    dbias = None if bias_dtype is None else s.new_empty(cols, dtype=bias_dtype)
    nbytes = lib.mcclx_layer_norm_workspace_bytes(q.handle, rows, cols)
    work = s.new_empty(nbytes, dtype=torch.uint8)
    a = L.Norm(dtype_code(s), param, rows, cols, 0.0, p, seed, offset, _ptr(weight), None, mean.data_ptr(), rstd.data_ptr(),
               None, None, None, sr.data_ptr(), dyr.data_ptr(), _ptr(ds), _ptr(dx), _ptr(dresidual), _ptr(dweight),
               _ptr(dbias), 0, 0, s_stride, dy_stride, ds_stride, work.data_ptr(), nbytes)
    L.check(lib.mcclx_layer_norm_backward(q.handle, _stream(q), C.byref(a)))
    return dx, dresidual, dweight, dbias


def layer_norm_forward(x, weight=None, bias=None, eps: float = 1e-5, queue=None):
    """(y, mean, rstd) of rows x: y = (x - mean) * rstd * weight + bias.  weight and bias have x's
    dtype or float32, or are None; mean and rstd = 1 / sqrt(variance + eps) are float32."""
    y, _, mean, rstd = _norm_forward(_q(queue), x, None, weight, bias, 0.0, 0, 0, eps, False)
    return y, mean, rstd


def _bias_dtype(with_bias: bool, bias_dtype, weight, x):
    return None if not with_bias else bias_dtype if bias_dtype is not None else x.dtype if weight is None else weight.dtype


def layer_norm_backward(dy, x, mean, rstd, weight=None, with_bias: bool = True, queue=None, *, bias_dtype=None,
                        with_x: bool = True, with_weight: bool = True):
    """(dx, dweight, dbias), None where not wanted; dweight is None without a weight too.  bias_dtype is the bias's where
    there is no weight to tell it (None: x's).  Sums over the rows are taken in the same order in every call; without dweight and
    dbias the pass is one launch."""
    dx, _, dweight, dbias = _norm_backward(_q(queue), dy, None, x, mean, rstd, weight, 0.0, 0, 0, with_x, False, with_weight,
                                           _bias_dtype(with_bias, bias_dtype, weight, x))
    return dx, dweight, dbias


def dropout_add_layer_norm_forward(x, residual, weight=None, bias=None, p: float = 0.0, seed: int = 0, offset: int = 0,
                                   eps: float = 1e-5, queue=None):
    """(y, s, mean, rstd): s = residual + dropout(x), y = layer_norm(s), in one pass.  y comes from the
    sum before it is rounded into s."""
    p, seed, offset = _mask(p, seed, offset)
    return _norm_forward(_q(queue), x, residual, weight, bias, p, seed, offset, eps, True)


def dropout_add_layer_norm_backward(dy, ds, s, mean, rstd, weight=None, p: float = 0.0, seed: int = 0, offset: int = 0,
                                    with_bias: bool = True, queue=None, *, bias_dtype=None, with_x: bool = True,
                                    with_residual: bool = True, with_weight: bool = True):
    """(dx, dresidual, dweight, dbias) from the gradients of y and of s (ds may be None), as in layer_norm_backward."""
    p, seed, offset = _mask(p, seed, offset)
    return _norm_backward(_q(queue), dy, ds, s, mean, rstd, weight, p, seed, offset, with_x, with_residual, with_weight,
                          _bias_dtype(with_bias, bias_dtype, weight, s))


# ---- dropout ----------------------------------------------------------------------

def dropout_forward(x, p: float, seed: int, offset: int = 0, residual=None, queue=None):
    """dropout(x), plus the residual where there is one.  What is kept depends on (seed, offset) and
    on an element's row and column, on nothing else; kept elements are scaled by the inverse of the share that is
    kept.  See mcclx_dropout in include/mcclx.h for the exact bits."""
    q = _q(queue)
    p, seed, offset = _mask(p, seed, offset)
    native = _reader()
    if native is not None:
        done = native._dropout(q.handle.value, q.device, x, residual, p, seed, offset)
        if done is not None:
            L.check(done[0])
            return done[1]
    xr, rows, cols, x_stride = _rows(q, x, "x")
    r_stride = 0
    if residual is not None:
        _same(x, residual, "residual")
        residual, _, _, r_stride = _rows(q, residual, "residual")
    out = _like(x)
    L.check(L.lib().mcclx_dropout(q.handle, _stream(q), dtype_code(x), rows, cols, xr.data_ptr(), x_stride, _ptr(residual),
                                  r_stride, out.data_ptr(), p, seed, offset))
    return out


def dropout_backward(dy, p: float, seed: int, offset: int = 0, queue=None):
    """The gradient of x: dropout of dy with the same mask.  (The residual's is dy itself.)"""
    return dropout_forward(dy, p, seed, offset, queue=queue)


class MaskStream:
    """Hands out a (seed, offset) for each use of dropout.  Ranks of one training run share the seed and
    differ in rank, which sits in the offset's upper bits; state_dict() is what a checkpoint keeps, and
    a run that continues from it draws the masks it would have drawn.  A stream that was given a rank keeps it whatever
    state it loads: all ranks may resume from one rank's checkpoint.  Without one (None: rank 0) it takes the state's."""

    def __init__(self, seed: int, rank: Optional[int] = None):
        if rank is not None and not 0 <= rank < 1 << 16:
            raise MCCLError(f"[MCCL] MaskStream: rank {rank} outside 0..65535")
        self.seed, self.rank, self.count = int(seed) & _M64, rank or 0, 0
        self._own_rank = rank is not None

    def next(self) -> Tuple[int, int]:
        offset = (self.rank << 48) | (self.count & ((1 << 48) - 1))
        self.count += 1
        return self.seed, offset

    def state_dict(self) -> dict:
        return {"seed": self.seed, "rank": self.rank, "count": self.count}

    def load_state_dict(self, state: dict) -> None:
        self.seed, self.count = state["seed"], state["count"]
        if not self._own_rank:
            self.rank = state["rank"]


# ---- the loss ------------------------------------------------------------------------

_REDUCTIONS = {"none": L.LOSS_NONE, "mean": L.LOSS_MEAN, "sum": L.LOSS_SUM}


def _loss_args(q, hidden, weight, target, lse, ignore_index, reduction):
    """The call's arguments and the tensors they point into, which have to outlive the call."""
    if weight.dim() != 2:
        raise MCCLError(f"[MCCL] weight: expected (vocabulary, width), got shape {tuple(weight.shape)}")
    h, tokens, width, h_stride = _rows(q, hidden, "hidden")
    w, vocab, wide, w_stride = _rows(q, weight, "weight")
    if width != wide:
        raise MCCLError(f"[MCCL] weight: rows of {wide} elements beside hidden's of {width}")
    if hidden.dtype != weight.dtype:
        raise MCCLError(f"[MCCL] weight: dtype {weight.dtype} beside {hidden.dtype}")
    _on_gpu(q, target, "target")
    if target.dtype != torch.int64 or target.shape != hidden.shape[:-1]:
        raise MCCLError(f"[MCCL] target: expected int64 of shape {tuple(hidden.shape[:-1])}, got {target.dtype} of {tuple(target.shape)}")
    if reduction not in _REDUCTIONS:
        raise MCCLError(f"[MCCL] linear_cross_entropy: reduction {reduction!r} unknown")
    target = target.contiguous()
    a = L.Loss(dtype_code(hidden), _REDUCTIONS[reduction], tokens, vocab, width, h.data_ptr(), w.data_ptr(), h_stride, w_stride,
               target.data_ptr(), int(ignore_index))
    a.lse = lse.data_ptr()
    return a, (h, w, target)


def linear_cross_entropy_forward(hidden, weight, target, ignore_index: int = -100, reduction: str = "mean", queue=None):
    """(loss, lse): softmax cross entropy of hidden @ weight.T, whose logits are never stored, and the
    logarithm of each token's sum of exponentials.  hidden is (..., width), weight (vocabulary, width),
    target (...) int64.  Targets equal to ignore_index have the loss 0 and do not count in the mean, which is NaN
    where none is left; a target outside the vocabulary makes its loss, and what its gradient reaches, NaN.  Both
    results are float32.  float32 matrices are multiplied with float32's precision, for values down to 2^-100 of the
    largest finite one of their matrix."""
    q = _q(queue)
    _on_gpu(q, hidden, "hidden")
    lse = hidden.new_empty(hidden.shape[:-1], dtype=torch.float32)
    a, keep = _loss_args(q, hidden, weight, target, lse, ignore_index, reduction)
    loss = torch.empty_like(lse) if reduction == "none" else lse.new_empty(())
    lib = L.lib()
    nbytes = lib.mcclx_linear_cross_entropy_workspace_bytes(q.handle, C.byref(a), 0)
    work = hidden.new_empty(nbytes, dtype=torch.uint8)
    a.loss, a.workspace, a.workspace_bytes = loss.data_ptr(), work.data_ptr(), nbytes
    L.check(lib.mcclx_linear_cross_entropy_forward(q.handle, _stream(q), C.byref(a)))
    return loss, lse


def linear_cross_entropy_backward(grad, hidden, weight, target, lse, ignore_index: int = -100, reduction: str = "mean",
                                  with_hidden: bool = True, with_weight: bool = True, queue=None):
    """(dhidden, dweight), None where not wanted, from the gradient of the loss (float32, of its shape) and the
    forward pass's lse.  The logits are computed again, for pieces of the vocabulary."""
    q = _q(queue)
    _on_gpu(q, hidden, "hidden")
    _stats(q, lse, target.numel(), "lse")
    a, keep = _loss_args(q, hidden, weight, target, lse, ignore_index, reduction)
    _on_gpu(q, grad, "grad")
    if grad.dtype != torch.float32 or grad.numel() != (target.numel() if reduction == "none" else 1):
        raise MCCLError(f"[MCCL] grad: expected float32 of the loss's shape, got {grad.dtype} of {tuple(grad.shape)}")
    grad = grad.contiguous()
    dhidden = _like(hidden) if with_hidden else None
    dweight = _like(weight) if with_weight else None
    lib = L.lib()
    nbytes = lib.mcclx_linear_cross_entropy_workspace_bytes(q.handle, C.byref(a), 1)
    work = hidden.new_empty(nbytes, dtype=torch.uint8)
    a.grad, a.dhidden, a.dweight = grad.data_ptr(), _ptr(dhidden), _ptr(dweight)
    a.workspace, a.workspace_bytes = work.data_ptr(), nbytes
    L.check(lib.mcclx_linear_cross_entropy_backward(q.handle, _stream(q), C.byref(a)))
    return dhidden, dweight


# ---- differentiable forms -----------------------------------------------------------

class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, queue):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps, queue)
        ctx.save_for_backward(x, mean, rstd, weight)
        ctx.bias_dtype, ctx.queue = bias.dtype if ctx.needs_input_grad[2] else None, queue
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, mean, rstd, weight = ctx.saved_tensors
        need = ctx.needs_input_grad
        return (*layer_norm_backward(dy, x, mean, rstd, weight, need[2], ctx.queue, bias_dtype=ctx.bias_dtype, with_x=need[0],
                                     with_weight=need[1]), None, None)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset, queue):
        ctx.mask, ctx.has_residual, ctx.queue = (p, seed, offset), residual is not None, queue
        return dropout_forward(x, p, seed, offset, residual, queue)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        dx = dropout_backward(dy, *ctx.mask, queue=ctx.queue) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.has_residual else None, None, None, None, None


class _Seam(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, p, seed, offset, eps, queue):
        y, s, mean, rstd = dropout_add_layer_norm_forward(x, residual, weight, bias, p, seed, offset, eps, queue)
        ctx.save_for_backward(s, mean, rstd, weight)
        ctx.mask, ctx.bias_dtype, ctx.queue = (p, seed, offset), bias.dtype if ctx.needs_input_grad[3] else None, queue
        ctx.set_materialize_grads(False)
        return y, s

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, ds):
        s, mean, rstd, weight = ctx.saved_tensors
        if dy is None:
            dy = torch.zeros_like(s)
        need = ctx.needs_input_grad
        return (*dropout_add_layer_norm_backward(dy, ds, s, mean, rstd, weight, *ctx.mask, need[3], ctx.queue, bias_dtype=ctx.bias_dtype,
                                                 with_x=need[0], with_residual=need[1], with_weight=need[2]),
                None, None, None, None, None)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, ignore_index, reduction, queue):
        loss, lse = linear_cross_entropy_forward(hidden, weight, target, ignore_index, reduction, queue)
        ctx.save_for_backward(hidden, weight, target, lse)
        ctx.rest = ignore_index, reduction, queue
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        hidden, weight, target, lse = ctx.saved_tensors
        ignore_index, reduction, queue = ctx.rest
        return (*linear_cross_entropy_backward(grad, hidden, weight, target, lse, ignore_index, reduction, ctx.needs_input_grad[0],
                                               ctx.needs_input_grad[1], queue), None, None, None, None)


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, queue=None) -> torch.Tensor:
    """Differentiable layer_norm_forward."""
    return _LayerNorm.apply(x, weight, bias, eps, queue)


def _next(p: float, masks: Optional[MaskStream], what: str) -> Tuple[int, int]:
    if masks is not None:
        return masks.next()
    if p:
        raise MCCLError(f"[MCCL] {what}: p > 0 needs a MaskStream")
    return 0, 0


def dropout(x, p: float, masks: Optional[MaskStream] = None, residual=None, queue=None) -> torch.Tensor:
    """Differentiable dropout_forward, with the next mask of `masks`."""
    return _Dropout.apply(x, residual, p, *_next(p, masks, "dropout"), queue)


def dropout_add_layer_norm(x, residual, weight=None, bias=None, p: float = 0.0, masks: Optional[MaskStream] = None,
                           eps: float = 1e-5, queue=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Differentiable (y, s): s = residual + dropout(x) with the next mask of `masks` (residual None: without the sum),
    y = layer_norm(s)."""
    return _Seam.apply(x, residual, weight, bias, p, *_next(p, masks, "dropout_add_layer_norm"), eps, queue)


def linear_cross_entropy(hidden, weight, target, ignore_index: int = -100, reduction: str = "mean", queue=None) -> torch.Tensor:
    """Differentiable linear_cross_entropy_forward: the loss alone."""
    return _LinearCrossEntropy.apply(hidden, weight, target, ignore_index, reduction, queue)
