"""Global norm of many gradients, and clipping."""
from __future__ import annotations

from array import array
from functools import lru_cache

import torch
from torch.autograd.graph import increment_version

from .. import _native as N

_DTYPES = {torch.float32: N.F32, torch.bfloat16: N.BF16, torch.float16: N.F16}
_NORMS = {1.0: 1, 2.0: 2, float("inf"): 0}


@lru_cache(maxsize=64)
def _workspace_bytes(count):
    n = N.c_i64(0)
    N.call("mib_clip_grad_norm_workspace", count, n)
    return n.value


def _dense(t):
    """Whether the tensor's elements fill one gapless range of memory (in any order of its dimensions)."""
    if t.is_contiguous():
        return True
    at = 1
    for s, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n != 1):
        if s != at:
            return False
        at *= n
    return True


def _gradients(tensors):
    if isinstance(tensors, torch.Tensor):
        tensors = [tensors]
    grads = []
    for t in tensors:
        if isinstance(t, torch.nn.Parameter) or (t.requires_grad and t.is_leaf):  # a weight: never scaled itself
            t = t.grad
            if t is None:
                continue
        grads.append(t)
    return grads


def _run(grads, max_norm, norm_type, eps, out):
    mode = _NORMS.get(float(norm_type))
    if mode is None:
        raise ValueError(f"norm_type must be 1, 2 or inf, got {norm_type}")
    if not grads:
        return torch.zeros(())
    index = grads[0].get_device()
    if index < 0:
        raise ValueError("gradients must be on a CUDA device")
    lists = [grads] if out is None or out is grads else [grads, out]
    types = []
    for group in lists:
        if any(t.get_device() != index for t in group):
            raise ValueError("gradients on more than one device")
        try:
            types.append(array("i", [_DTYPES[t.dtype] for t in group]))
        except KeyError as e:
            raise ValueError(f"gradients must be float32, bfloat16 or float16, got {e.args[0]}") from None
        if not all(t.is_contiguous() or _dense(t) for t in group):
            raise ValueError("gradients must be dense in memory (no gaps between elements)")
    if len(lists) == 2:
        if len(out) != len(grads):
            raise ValueError(f"out holds {len(out)} tensors, expected {len(grads)}")
        if any(g.shape != o.shape or not (g.is_contiguous() and o.is_contiguous() or g.stride() == o.stride())
               for g, o in zip(grads, out)):
            raise ValueError("out must have the gradients' shapes and strides")
    ptrs = [array("q", [t.data_ptr() for t in g]) for g in lists]
    if out is not None and len(set(ptrs[-1])) != len(out):
        used = [t.data_ptr() for t in lists[-1] if t.numel()]
        if len(set(used)) != len(used):
            raise ValueError("the same gradient is listed twice")
    numel = array("q", [t.numel() for t in grads])
    nbytes = _workspace_bytes(len(grads))
    first = grads[0]
    ws, norm = first.new_empty(nbytes, dtype=torch.uint8), first.new_empty((), dtype=torch.float32)
    at = lambda a: a.buffer_info()[0]  # noqa: E731
    N.launch("mib_clip_grad_norm", index, at(ptrs[0]), None if out is None else at(ptrs[-1]), at(numel), at(types[0]),
             None if out is None else at(types[-1]), len(grads), mode, max_norm, eps, norm.data_ptr(), ws.data_ptr(), nbytes)
    if out is not None:  # written behind autograd's back: what a graph has saved of them is gone
        increment_version(out)
    return norm


@torch.no_grad()
def grad_norm(tensors, norm_type=2.0):
    """Norm (1, 2 or inf) of all gradients together, a 0-d fp32 tensor.  ``tensors``: gradients, or parameters and
    other leaf tensors that require a gradient (their ``.grad`` is taken; those without one are skipped)."""
    return _run(_gradients(tensors), 0.0, norm_type, 0.0, None)


@torch.no_grad()
def clip_grad_norm_(tensors, max_norm, norm_type=2.0, *, out=None, eps=1e-6):
    """Multiply all gradients by ``min(1, max_norm / (norm + eps))`` and return the norm before that (0-d, fp32).

    ``tensors`` as in ``grad_norm``.  In place, or into ``out``: one tensor per gradient, of its shape and strides and
    any of the three types (fp32 copies of fp16 gradients, for instance); the gradients then stay as they are.  Nothing
    waits for the GPU; a non-finite norm shows in the returned value and, as in the formula, in the gradients."""
    if not 0.0 <= max_norm < float("inf"):
        raise ValueError("max_norm must be non-negative and finite")
    if not 0.0 <= eps < float("inf"):
        raise ValueError("eps must be non-negative")
    grads = _gradients(tensors)
    return _run(grads, max_norm, norm_type, eps, grads if out is None else list(out))
