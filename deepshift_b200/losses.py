"""Softmax cross entropy of a linear head over a large vocabulary, without its logits.

``linear_cross_entropy(hidden, weight, target)`` is ``F.cross_entropy(hidden @ weight.T, target)`` with the logits computed tile
by tile on the tensor cores and never stored: forward, each tile leaves a maximum and a sum for each row; backward, the logits are
computed again a piece of the vocabulary at a time, whose gradient (at most 256 MB in 16 bits) makes that piece's part of both
gradients.  Differentiable in ``hidden`` and ``weight``.  Runs on torch's current stream; scratch comes from torch's allocator.
No counterpart in the reference.
"""
import torch

from . import _ffi
from .kernels import _stream_ptr

_TYPES = {torch.bfloat16: _ffi.T_BF16, torch.float16: _ffi.T_F16}
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}

MAX_ROWS, MAX_WIDTH, MAX_VOCABULARY = 1 << 24, 1 << 20, 1 << 24


def _check(hidden, weight, target, reduction):
    if reduction not in _REDUCTIONS:
        raise ValueError("reduction must be none, mean or sum, got %r" % (reduction,))
    if not hidden.is_cuda:
        raise RuntimeError("hidden must be a CUDA tensor")
    if hidden.dtype not in _TYPES or weight.dtype != hidden.dtype:
        raise RuntimeError("hidden and weight must both be bfloat16 or float16, got %s and %s" % (hidden.dtype, weight.dtype))
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.size(-1) != weight.size(1):
        raise RuntimeError("hidden must be [..., d] and weight [v, d], got %s and %s" % (tuple(hidden.shape), tuple(weight.shape)))
    if target.shape != hidden.shape[:-1] or target.dtype not in (torch.int64, torch.int32):
        raise RuntimeError("target must be int64 %s, got %s of %s" % (tuple(hidden.shape[:-1]), target.dtype, tuple(target.shape)))
    if weight.device != hidden.device or target.device != hidden.device:
        raise RuntimeError("hidden, weight and target must be on one device")
    v, d = weight.shape
    if target.numel() > MAX_ROWS or not 1 <= d <= MAX_WIDTH or not 1 <= v <= MAX_VOCABULARY:
        raise RuntimeError("at most %d rows of 1 .. %d and a vocabulary of 1 .. %d, got %d, %d and %d"
                           % (MAX_ROWS, MAX_WIDTH, MAX_VOCABULARY, target.numel(), d, v))


def _call(hidden, weight, target, ignore_index, reduction, backward):
    """The structure of a call, and its scratch."""
    a = _ffi.Loss()
    a.rows, a.d, a.v = hidden.size(0), weight.size(1), weight.size(0)
    a.type, a.reduction, a.ignore_index = _TYPES[hidden.dtype], reduction, ignore_index
    a.hidden, a.weight, a.target = hidden.data_ptr(), weight.data_ptr(), target.data_ptr()
    n = _ffi.lib().ds_loss_bytes(a.rows, a.d, a.v, backward, int(bool((a.hidden or 0) & 15 or a.weight & 15)))
    scratch = torch.empty(n, dtype=torch.uint8, device=hidden.device)
    a.scratch, a.scratch_bytes = scratch.data_ptr(), n
    return a, scratch


def _forward(hidden, weight, target, ignore_index, reduction):
    a, scratch = _call(hidden, weight, target, ignore_index, reduction, 0)
    each, lse = torch.empty((2, a.rows), dtype=torch.float32, device=hidden.device).unbind()
    whole = torch.empty(2, dtype=torch.float32, device=hidden.device) if reduction else None
    a.each, a.lse = each.data_ptr(), lse.data_ptr()
    if reduction:
        a.loss, a.count = whole.data_ptr(), whole.data_ptr() + 4
    with torch.cuda.device(hidden.device):
        _ffi.check(_ffi.lib().ds_loss_forward(a, _stream_ptr(hidden.device)), "linear_cross_entropy")
    return each, lse, whole


class _Loss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, ignore_index, reduction):
        each, lse, whole = _forward(hidden, weight, target, ignore_index, reduction)
        ctx.save_for_backward(hidden, weight, target, lse, whole)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        return whole[0] if reduction else each.clone()

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        hidden, weight, target, lse, whole = ctx.saved_tensors
        grad = grad.contiguous()
        a, scratch = _call(hidden, weight, target, ctx.ignore_index, ctx.reduction, 1)
        a.lse, a.grad = lse.data_ptr(), grad.data_ptr()
        if ctx.reduction:
            a.count = whole.data_ptr() + 4
        dhidden = dweight = None
        if ctx.needs_input_grad[0]:
            dhidden = torch.empty_like(hidden)
            a.dhidden = dhidden.data_ptr()
        if ctx.needs_input_grad[1]:
            dweight = torch.empty_like(weight)
            a.dweight = dweight.data_ptr()
        with torch.cuda.device(hidden.device):
            _ffi.check(_ffi.lib().ds_loss_backward(a, _stream_ptr(hidden.device)), "linear_cross_entropy (backward)")
        return dhidden, dweight, None, None, None


def linear_cross_entropy(hidden, weight, target, ignore_index=-100, reduction="mean"):
    """Cross entropy of ``hidden @ weight.T`` against ``target`` as fp32: the mean or the sum over the rows whose target is not
    ``ignore_index``, or (``reduction="none"``) each row's, 0 for those.

    ``hidden`` [..., d] and ``weight`` [v, d] are bfloat16 or float16, both the same; ``target`` is integer, of the shape of
    ``hidden`` without its last dimension.  Sums are fp32.  The gradient of the logits is rounded to 16 bits once before it is
    multiplied (in float16 it is scaled to use the whole range).  A target outside 0 .. v - 1 makes its row's loss NaN, and
    the gradients that it enters; the mean over no rows at all is NaN and its gradients are 0."""
    _check(hidden, weight, target, reduction)
    code = _REDUCTIONS[reduction]
    shape = target.shape
    rows = hidden.reshape(-1, hidden.size(-1)).contiguous()
    weight = weight.contiguous()
    flat = target.reshape(-1).to(torch.int64).contiguous()
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        loss = _Loss.apply(rows, weight, flat, int(ignore_index), code)
    else:
        each, _, whole = _forward(rows, weight, flat, int(ignore_index), code)
        loss = whole[0] if code else each
    return loss if code else loss.view(shape)
