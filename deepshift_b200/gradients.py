"""The global norm of many gradients, and their clipping, on the GPU and without a synchronisation.

``clip_norm`` reads every tensor of a list, forms sqrt(sum of all squares) and multiplies each by min(1, max_norm / (norm +
1e-6)), in place or into tensors given; ``clip_grad_norm_`` does so for the gradients of parameters, as
``torch.nn.utils.clip_grad_norm_`` with the 2-norm.  Two kernels for up to 512 tensors.  The sums are formed in a fixed order:
the same gradients give the same norm, bit for bit.  No counterpart in the reference.
"""
import ctypes
import math

import torch

from . import _ffi
from .adapters import TYPES
from .kernels import _stream_ptr


def _flat(t):
    """Whether a tensor's elements fill a stretch of memory, in whatever order."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != want:
            return False
        want *= size
    return True


def _run(tensors, to, max_norm, what):
    """One call of the library; ``to``: None for the norm alone."""
    device = tensors[0].device
    if device.type != "cuda":
        raise RuntimeError("gradients must be CUDA tensors")
    table, places = [], set()
    for i, t in enumerate(tensors):
        if t.layout is not torch.strided or t.dtype not in TYPES:
            raise RuntimeError("gradients must be dense, float32, bfloat16 or float16, got %s" % t.dtype)
        if t.device != device:
            raise RuntimeError("all gradients must be on one device")
        if not _flat(t):
            raise RuntimeError("a gradient must fill its memory without gaps")
        n, kind = t.numel(), TYPES[t.dtype]
        if to is None:
            table += (t.data_ptr(), 0, n, kind)
            continue
        o = to[i]
        if o is not t:
            if o.dtype not in TYPES or o.device != device:
                raise RuntimeError("out must be float32, bfloat16 or float16, on the gradients' device")
            if o.shape != t.shape or (o.stride() != t.stride() and not (o.is_contiguous() and t.is_contiguous())):
                raise RuntimeError("out must have the shapes and layouts of the gradients")
        at = o.data_ptr()
        if n:
            if at in places:
                raise RuntimeError("the same memory twice among the places that are written")
            places.add(at)
        table += (t.data_ptr(), at, n, kind | TYPES[o.dtype] << 32)
    norm = torch.empty((), dtype=torch.float32, device=device)
    lib = _ffi.lib()
    nbytes = lib.ds_clip_bytes(len(tensors))
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
    with torch.cuda.device(device):
        # an entry of ds_tensor_t is four words: the last holds both types
        _ffi.check(lib.ds_clip_norm((ctypes.c_int64 * len(table))(*table), len(tensors), max_norm, norm.data_ptr(),
                                    scratch.data_ptr(), nbytes, _stream_ptr(device)), what)
    return norm


def clip_norm(tensors, max_norm, out=None):
    """Scales ``tensors`` (float32, bfloat16, float16, mixed, of any shapes, on one GPU) so that their norm together is at most
    ``max_norm``; returns the norm before that as a float32 tensor on the GPU.

    ``out``: where the scaled values go, one tensor for each of ``tensors``, of its shape and layout and of any of the three
    types; None: in place.  ``max_norm = inf`` leaves the values as they are.  A norm that is NaN makes them NaN, an infinite
    one 0 (and NaN where they are infinite).  Empty tensors count for nothing."""
    tensors = list(tensors)
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError("max_norm must be >= 0, got %r" % max_norm)
    to = tensors if out is None else list(out)
    if len(to) != len(tensors):
        raise RuntimeError("%d tensors and %d places for them" % (len(tensors), len(to)))
    return _run(tensors, to, max_norm, "clip_norm") if tensors else torch.zeros(())


def global_norm(tensors):
    """The norm of all ``tensors`` together, as ``clip_norm`` forms it; changes nothing."""
    tensors = list(tensors)
    return _run(tensors, None, math.inf, "global_norm") if tensors else torch.zeros(())


def clip_grad_norm_(parameters, max_norm):
    """``clip_norm`` of the gradients of ``parameters`` (a tensor or an iterable; those without a gradient are left out), in
    place.  Returns their norm."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return clip_norm([p.grad for p in parameters if p.grad is not None], max_norm)
