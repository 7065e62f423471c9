"""Token embedding with a scale, and its gradient by sorted tokens."""
from __future__ import annotations

from functools import lru_cache

import torch
import torch.nn as nn
from torch.autograd.graph import increment_version

from .. import _native as N

_DTYPES = {torch.float32: N.F32, torch.bfloat16: N.BF16, torch.float16: N.F16}
_INTS = {torch.int32: 0, torch.int64: 1}


@lru_cache(maxsize=256)
def _workspace_bytes(n, vocab, hidden):
    b = N.c_i64(0)
    N.call("mib_embedding_grad_workspace", n, vocab, hidden, b)
    return b.value


def _check_ids(ids, index):
    """(ids, 1 if they are int64): dense, on CUDA device ``index``."""
    wide = _INTS.get(ids.dtype)
    if wide is None:
        raise ValueError(f"ids must be int32 or int64, got {ids.dtype}")
    if ids.get_device() != index:
        raise ValueError(f"ids is on {ids.device}, the embedding on cuda:{index}")
    return (ids if ids.is_contiguous() else ids.contiguous()), wide


def _lookup(ids, weight, scale):
    index = weight.get_device()
    if index < 0:
        raise ValueError("the embedding must be on a CUDA device")
    dtype = _DTYPES.get(weight.dtype)
    if dtype is None:
        raise ValueError(f"the embedding must be float32, bfloat16 or float16, got {weight.dtype}")
    shape = weight.shape
    if len(shape) != 2 or not shape[0] or not shape[1]:
        raise ValueError("the embedding must be (rows, columns) and non-empty")
    vocab, hidden = shape
    ld, unit = weight.stride()
    if vocab == 1:
        ld = hidden
    if hidden > 1 and unit != 1 or ld < hidden:
        raise ValueError("the embedding's rows must be dense")
    ids, wide = _check_ids(ids, index)
    out = weight.new_empty((*ids.shape, hidden))
    n = ids.numel()
    if n:
        N.launch("mib_embedding_lookup", index, ids.data_ptr(), wide, n, weight.data_ptr(), dtype, vocab, hidden, ld,
                 scale, out.data_ptr())
    return out


def embedding_scaled_grad(ids, grad_output, num_embeddings, scale=1.0, *, padding_idx=None, out=None,
                          accumulate=False):
    """Gradient of ``embedding_scaled`` over its table: ``dW[v] = scale * sum of grad_output[i] with ids[i] = v``.

    The sums are fp32, in token order (the same bits on every call).  Returns a dense (num_embeddings, H) tensor of
    ``grad_output``'s type; ``out`` takes it instead (that type or fp32, rows dense).  With ``accumulate`` the sums are
    added to ``out`` and only the rows of tokens that occur are touched.  ``padding_idx``'s tokens add nothing, nor do
    ids outside the table."""
    index = grad_output.get_device()
    if index < 0:
        raise ValueError("grad_output must be on a CUDA device")
    dtype = _DTYPES.get(grad_output.dtype)
    if dtype is None:
        raise ValueError(f"grad_output must be float32, bfloat16 or float16, got {grad_output.dtype}")
    shape = grad_output.shape
    if shape[:-1] != ids.shape or len(shape) != ids.dim() + 1 or shape[-1] < 1:
        raise ValueError(f"grad_output has shape {tuple(shape)}, expected {tuple(ids.shape)} + (H,)")
    if num_embeddings < 1:
        raise ValueError("num_embeddings must be positive")
    if padding_idx is None:
        padding_idx = -1
    elif not 0 <= padding_idx < num_embeddings:
        raise ValueError("padding_idx must be a row of the table")
    hidden = shape[-1]
    ld_out, out_dtype, given = hidden, dtype, out
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        out = grad_output.new_empty((num_embeddings, hidden))
    else:
        out_dtype = _DTYPES.get(out.dtype)
        if out.shape != (num_embeddings, hidden) or out.get_device() != index or out_dtype not in (dtype, N.F32):
            raise ValueError("out must be (num_embeddings, H) on grad_output's device, of its type or float32")
        if num_embeddings > 1:
            ld_out = out.stride(0)
        if hidden > 1 and out.stride(1) != 1 or ld_out < hidden:
            raise ValueError("out's rows must be dense and apart")
        if N.overlap(out, grad_output) or N.overlap(out, ids):
            raise ValueError("out shares memory with grad_output or ids")
    ids, wide = _check_ids(ids, index)
    n = ids.numel()
    if n == 0:
        return out if accumulate else out.zero_()
    g, ld = grad_output, hidden
    if not g.is_contiguous():
        g = g.detach()
        g = g if g.dim() == 2 else g.reshape(n, hidden)
        if hidden > 1 and g.stride(1) != 1 or n > 1 and g.stride(0) < hidden:
            g = g.contiguous()
        ld = g.stride(0) if n > 1 else hidden
    nbytes = _workspace_bytes(n, num_embeddings, hidden)
    ws = g.new_empty(nbytes, dtype=torch.uint8)
    N.launch("mib_embedding_grad", index, ids.data_ptr(), wide, n, g.data_ptr(), dtype, ld, num_embeddings, hidden, scale,
             padding_idx, out.data_ptr(), out_dtype, ld_out, 1 if accumulate else 0, ws.data_ptr(), nbytes)
    if given is not None:  # written behind autograd's back: what a graph has saved of it is gone
        increment_version(out)
    return out


class EmbeddingScaledRunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.args = (weight.shape[0], scale, padding_idx)
        return _lookup(ids, weight.detach(), scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output):
        (ids,), (rows, scale, padding_idx) = ctx.saved_tensors, ctx.args
        return None, embedding_scaled_grad(ids, grad_output, rows, scale, padding_idx=padding_idx), None, None


def embedding_scaled(ids, weight, scale=1.0, padding_idx=None):
    """``scale * weight[ids]``, rounded once to ``weight``'s type (fp32, bf16 or fp16).  Differentiable in ``weight``;
    ``padding_idx``'s tokens add nothing to its gradient.  An id outside the table gives a row of NaN."""
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise ValueError("padding_idx must be a row of the table")
    if weight.requires_grad and torch.is_grad_enabled():
        return EmbeddingScaledRunc.apply(ids, weight, float(scale), padding_idx)
    return _lookup(ids, weight, scale)


class EmbeddingScaled(nn.Module):
    """Token embedding ``scale * weight[ids]`` in front of crossbar layers (a table lookup: it has no crossbar).

    ``scale`` is a constant factor, such as ``sqrt(embedding_dim)``."""

    def __init__(self, num_embeddings: int, embedding_dim: int, scale: float = 1.0, padding_idx=None, device=None,
                 dtype=torch.float32):
        super().__init__()
        if padding_idx is not None and not 0 <= padding_idx < num_embeddings:
            raise ValueError("padding_idx must be a row of the table")
        self.num_embeddings, self.embedding_dim, self.scale = num_embeddings, embedding_dim, scale
        self.padding_idx = padding_idx
        self.weight = nn.Parameter(torch.empty((num_embeddings, embedding_dim), device=device, dtype=dtype))
        self.reset_parameters()

    def reset_parameters(self) -> None:
        nn.init.normal_(self.weight, std=0.02)
        if self.padding_idx is not None:
            with torch.no_grad():
                self.weight[self.padding_idx].zero_()

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return embedding_scaled(ids, self.weight, self.scale, self.padding_idx)
