"""Losses on the logits of a language model, and token log-probabilities.

``logits`` is (..., V), fp32, bf16 or fp16, on a CUDA device; ``targets`` holds the column of each row's token
(shape ``logits.shape[:-1]``, int32 or int64), ``ignore_index`` where a row takes no part (prompt and padding): such a
row's logits are not read, its log-probability is 0 and its gradient zero.  A target outside the vocabulary gives NaN.
A call takes fewer than 2^21 rows.

Sequences are the rows of a (B, T) batch of targets, or, with ``cu_seqlens`` (S + 1 non-decreasing row offsets),
ragged ones packed in one list of rows.

``policy_loss`` and ``preference_loss`` are differentiable in ``logits``: the forward call keeps 16 bytes of each row, the
backward call forms the gradient from them and the logits, with what multiplies the loss (a loss scale, say) before the
gradient's only rounding to their type.  ``policy_loss_grad`` and ``preference_loss_grad`` return the loss and that gradient without
autograd, into ``out`` if given: ``out=logits`` overwrites the logits and saves the gradient's memory.
"""
from __future__ import annotations

from collections import namedtuple
from functools import lru_cache

import torch
from torch.autograd.graph import increment_version

from .. import _native as N

_DTYPES = {torch.float32: N.F32, torch.bfloat16: N.BF16, torch.float16: N.F16}
_INTS = {torch.int32: 0, torch.int64: 1}
_REDUCTIONS = {"token": 0, "sequence": 1, "sum": 2}
_PER = {None: None, "token": True, "sequence": False}
_KINDS = {"sigmoid": 0, "hinge": 1, "squared": 2}

#: loss, per-token log-probabilities, weighted KL term (without its coefficient), weighted fraction of clipped tokens
PolicyLoss = namedtuple("PolicyLoss", "loss logps kl clip_fraction")
#: loss, beta times each pair's summed log ratio (chosen, rejected), per-token log-probabilities
PreferenceLoss = namedtuple("PreferenceLoss", "loss chosen_rewards rejected_rewards logps")


def _layout(t):
    """Row addressing of a (..., V) tensor with unit column stride in at most two levels, or None."""
    shape, strides = t.shape, t.stride()
    cols = shape[-1]
    if t.is_contiguous():
        return N.OutLayout(max(1, t.numel() // cols), 0, cols, 1)
    merged = []
    for n, s in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if n == 1:
            continue
        if merged and s == merged[-1][0] * merged[-1][1]:
            merged[-1] = (merged[-1][0] * n, merged[-1][1])
        else:
            merged.append((n, s))
    if len(merged) > 2 or (cols != 1 and strides[-1] != 1):
        return None
    n, s = merged[0] if merged else (1, cols)
    if n > 1 and s < cols:
        return None
    return N.OutLayout(max(1, n), merged[1][1] if len(merged) == 2 else 0, s, 1)


def _ints(t, what, index):
    """(t, 1 if it is int64): dense, on CUDA device ``index``."""
    wide = _INTS.get(t.dtype)
    if wide is None:
        raise ValueError(f"{what} must be int32 or int64, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{what} is on {t.device}, the logits on cuda:{index}")
    return (t if t.is_contiguous() else t.contiguous()), wide


def _floats(t, what, shape, index):
    if t.shape != shape:
        raise ValueError(f"{what} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.get_device() != index:
        raise ValueError(f"{what} is on {t.device}, the logits on cuda:{index}")
    if t.dtype is torch.float32 and t.is_contiguous():
        return t
    return t.detach().to(torch.float32).contiguous()


class _Rows:
    """The checked rows of one call: the native description and the tensors it points into."""
    __slots__ = ("n", "sequences", "logits", "targets", "cu", "index", "spec")

    def __init__(self, logits, targets, temperature, ignore_index, cu_seqlens=None):
        index = logits.get_device()
        if index < 0:
            raise ValueError("logits must be on a CUDA device")
        dtype = _DTYPES.get(logits.dtype)
        if dtype is None:
            raise ValueError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
        shape = logits.shape
        if len(shape) < 1 or shape[-1] < 1:
            raise ValueError("logits must be (..., V) with V >= 1")
        if targets.shape != shape[:-1]:
            raise ValueError(f"targets has shape {tuple(targets.shape)}, expected {tuple(shape[:-1])}")
        if not 1e-30 <= temperature < 1e30:
            raise ValueError("temperature must be positive, from 1e-30 to 1e30")
        layout = _layout(logits)
        if layout is None:
            logits = logits.detach().contiguous()
            layout = _layout(logits)
        targets, wide = _ints(targets, "targets", index)
        n = targets.numel()
        cu, cu_wide, sequences, per = None, 0, 0, 0
        if cu_seqlens is not None:
            if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
                raise ValueError("cu_seqlens must hold the S + 1 row offsets of S sequences")
            cu_seqlens, cu_wide = _ints(cu_seqlens, "cu_seqlens", index)
            cu, sequences = cu_seqlens.data_ptr(), cu_seqlens.numel() - 1
        elif len(shape) > 2:
            per = shape[-2]
            sequences = n // per if per else 0
        self.n, self.sequences, self.index = n, sequences, index
        self.logits, self.targets, self.cu = logits, targets, cu_seqlens
        self.spec = N.TokenRows(logits.data_ptr(), targets.data_ptr(), cu, n, shape[-1], layout, ignore_index, sequences,
                                per, temperature, dtype, wide, cu_wide, 0)

    def empty(self, shape):
        return self.logits.new_empty(shape, dtype=torch.float32)

    def workspace(self):
        nbytes = _workspace_bytes(self.n, self.spec.cols, self.sequences)
        return self.logits.new_empty(nbytes, dtype=torch.uint8), nbytes

    def gradient(self, out, *read):
        """The gradient's tensor and row addressing; ``read``: what the call reads beside the rows."""
        a = self.logits
        if out is None:
            out = a.new_empty(a.shape)
            return out, _layout(out)
        if out.shape != a.shape or out.dtype != a.dtype or out.get_device() != self.index:
            raise ValueError("out must have the logits' shape, type and device")
        layout = _layout(out)
        if layout is None or not _apart(layout, self.n, out.shape[-1]):
            raise ValueError("out needs a unit column stride and rows that do not overlap")
        if a.data_ptr() == out.data_ptr():
            if a.stride() != out.stride() and self.n > 1:
                raise ValueError("out overlaps the logits without being the same rows")
        elif N.overlap(a, out):
            raise ValueError("out overlaps the logits without being the same rows")
        if any(t is not None and N.overlap(out, t) for t in (self.targets, self.cu, *read)):
            raise ValueError("out shares memory with another argument")
        return out, layout


def _apart(layout, rows, cols):
    """Whether no two rows of at most two levels share an element: either level may be the outer one."""
    inner, step, jump = layout.rows_per_group, layout.row_stride, layout.group_stride
    if rows <= inner:
        return True
    return jump >= (inner - 1) * step + cols or cols <= jump and step >= (rows // inner - 1) * jump + cols


def _address(t):
    return None if t is None else t.data_ptr()


@lru_cache(maxsize=256)
def _workspace_bytes(rows, cols, sequences):
    n = N.c_i64(0)
    N.call("mib_token_loss_workspace", rows, cols, sequences, n)
    return n.value


# ---- log-probabilities ---------------------------------------------------------------------------------
class TokenLogprobsRunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, temperature, ignore_index):
        rows = _Rows(logits, targets, temperature, ignore_index)
        keep = ctx.needs_input_grad[0]
        logps, stats = _token_logps(rows, keep)
        if keep:
            ctx.save_for_backward(logits, targets, stats)
            ctx.args = (temperature, ignore_index)
        return logps

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_logps):
        logits, targets, stats = ctx.saved_tensors
        rows = _Rows(logits, targets, *ctx.args)
        grad, layout = rows.gradient(None)
        if rows.n:
            g = _floats(grad_logps, "the gradient", targets.shape, rows.index)
            N.launch("mib_token_logps_grad", rows.index, rows.spec, stats.data_ptr(), g.data_ptr(), grad.data_ptr(), layout)
        return grad, None, None, None


def _token_logps(rows, keep_stats):
    logps = rows.empty(rows.targets.shape)
    stats = rows.empty((rows.n, 4)) if keep_stats else None
    if rows.n:
        N.launch("mib_token_logps", rows.index, rows.spec, logps.data_ptr(), _address(stats))
    return logps, stats


def token_logprobs(logits, targets, *, temperature=1.0, ignore_index=-100):
    """log softmax(logits / temperature) at each row's target, fp32 (0 at ignored rows).  Differentiable in ``logits``."""
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobsRunc.apply(logits, targets, float(temperature), int(ignore_index))
    return _token_logps(_Rows(logits, targets, float(temperature), int(ignore_index)), False)[0]


# ---- policy loss ---------------------------------------------------------------------------------------
def _policy(logits, targets, old_logps, advantages, ref_logps, clip_low, clip_high, kl_coef, cu_seqlens, reduction,
            temperature, ignore_index, advantages_per, want_grad, out):
    rows = _Rows(logits, targets, float(temperature), int(ignore_index), cu_seqlens)
    mode = _REDUCTIONS.get(reduction)
    if mode is None:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    clip_high = clip_low if clip_high is None else clip_high
    if not (0.0 <= clip_low <= 1.0 and 0.0 <= clip_high < float("inf")):
        raise ValueError("clip bounds must be non-negative and finite, the lower one at most 1")
    if not 0.0 <= kl_coef < float("inf"):
        raise ValueError("kl_coef must be non-negative")
    if kl_coef > 0.0 and ref_logps is None:
        raise ValueError("the KL term needs ref_logps")
    if mode == 1 and rows.sequences < 1 and rows.n:
        raise ValueError("the sequence mean needs a (B, T) batch or cu_seqlens")
    index, shape = rows.index, targets.shape
    old = _floats(old_logps, "old_logps", shape, index)
    if advantages_per not in _PER:
        raise ValueError(f'advantages_per must be "token", "sequence" or None, got {advantages_per!r}')
    per_token = _PER[advantages_per]
    if per_token is None:  # a list with an entry per sequence is that, even where there are as many rows
        per_token = advantages.shape == shape and (cu_seqlens is None or len(shape) != 1 or shape[0] != rows.sequences)
    if advantages.shape != shape if per_token else rows.sequences < 1 or advantages.numel() != rows.sequences:
        raise ValueError(f"advantages has shape {tuple(advantages.shape)}, expected {tuple(shape)} or one per sequence "
                         f"({rows.sequences})")
    adv = _floats(advantages, "advantages", advantages.shape, index)
    ref = None if ref_logps is None else _floats(ref_logps, "ref_logps", shape, index)
    grad, layout = rows.gradient(out, old, adv, ref) if want_grad else (None, None)
    logps, res = rows.empty(shape), rows.empty(3)
    ws, nbytes = rows.workspace() if rows.n else (None, 0)
    if ws is None:
        res.zero_()
    else:
        spec = N.PolicySpec(clip_low, clip_high, kl_coef, mode, 0 if per_token else 1)
        N.launch("mib_policy_loss", index, rows.spec, spec, old.data_ptr(), adv.data_ptr(), _address(ref), res.data_ptr(),
                 logps.data_ptr(), _address(grad), layout, ws.data_ptr(), nbytes)
    if out is not None:  # written behind autograd's back: what a graph has saved of it is gone
        increment_version(out)
    loss, kl, clipped = res.unbind(0)
    return PolicyLoss(loss, logps, kl, clipped), grad, ws


class _LossRunc(torch.autograd.Function):
    """A loss that depends on each row through its log-probability: backward needs the logits and the rows' statistics and
    coefficients, which ``evaluate`` leaves in its workspace."""

    @staticmethod
    def forward(ctx, logits, targets, cu_seqlens, temperature, ignore_index, evaluate):
        result, ctx.space = evaluate(logits)
        ctx.spent = False
        ctx.save_for_backward(logits, targets, cu_seqlens)
        ctx.args = (temperature, ignore_index)
        ctx.mark_non_differentiable(*result[1:])
        loss = result[0]
        if loss._is_view():  # one of several views of a buffer: autograd would refuse to change it in place
            loss = loss.new_empty(0).set_(loss)
        return (loss, *result[1:])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss, *_):
        space, ctx.space, spent, ctx.spent = ctx.space, None, ctx.spent, True
        if spent:
            raise RuntimeError("the loss's row statistics were already given back: a second backward pass needs a second "
                               "forward pass")
        logits, targets, cu_seqlens = ctx.saved_tensors
        rows = _Rows(logits, targets, *ctx.args, cu_seqlens)
        grad, layout = rows.gradient(None)
        if rows.n:
            factor = grad_loss.to(torch.float32).contiguous()
            N.launch("mib_loss_grad", rows.index, rows.spec, space.data_ptr(), space.numel(), factor.data_ptr(), grad.data_ptr(),
                     layout)
        return grad, None, None, None, None, None


def policy_loss(logits, targets, old_logps, advantages, ref_logps=None, *, clip_low=0.2, clip_high=None, kl_coef=0.0,
                cu_seqlens=None, reduction="token", temperature=1.0, ignore_index=-100, advantages_per=None):
    """Clipped policy loss with a KL term to a reference policy; returns a ``PolicyLoss``.

    Per token, with ``lp`` its log-probability, ``ratio = exp(lp - old_logps)`` and ``d = ref_logps - lp``:
    ``-min(ratio A, clamp(ratio, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(d) - d - 1)``.  ``reduction``: "token"
    (mean over the tokens that take part), "sequence" (mean over the sequences that have such tokens of their token
    means) or "sum".  ``advantages``: one per token or one per sequence, as their number says, or as ``advantages_per``
    ("token" or "sequence") does: with ``cu_seqlens`` and as many sequences as rows they are taken per sequence, which
    differs where a sequence is empty.  ``clip_high`` defaults to ``clip_low``.
    Without a token that takes part the loss is 0."""
    def evaluate(x):
        return _policy(x, targets, old_logps, advantages, ref_logps, clip_low, clip_high, kl_coef, cu_seqlens,
                       reduction, temperature, ignore_index, advantages_per, False, None)[::2]
    if logits.requires_grad and torch.is_grad_enabled():
        return PolicyLoss(*_LossRunc.apply(logits, targets, cu_seqlens, float(temperature), int(ignore_index), evaluate))
    return evaluate(logits)[0]


def policy_loss_grad(logits, targets, old_logps, advantages, ref_logps=None, *, clip_low=0.2, clip_high=None,
                     kl_coef=0.0, cu_seqlens=None, reduction="token", temperature=1.0, ignore_index=-100,
                     advantages_per=None, out=None):
    """``policy_loss`` and the gradient of its loss over the logits, in their type: ``(PolicyLoss, grad)``."""
    return _policy(logits, targets, old_logps, advantages, ref_logps, clip_low, clip_high, kl_coef, cu_seqlens,
                   reduction, temperature, ignore_index, advantages_per, True, out)[:2]


# ---- preference loss -----------------------------------------------------------------------------------
def _preference(logits, targets, ref_logps, cu_seqlens, beta, label_smoothing, margin, kind, average, temperature,
                ignore_index, want_grad, out):
    rows = _Rows(logits, targets, float(temperature), int(ignore_index), cu_seqlens)
    mode = _KINDS.get(kind)
    if mode is None:
        raise ValueError(f"kind must be one of {sorted(_KINDS)}, got {kind!r}")
    if not 0.0 <= label_smoothing <= 0.5 or (mode != 0 and label_smoothing):
        raise ValueError("label_smoothing must be in [0, 0.5], and 0 except for the sigmoid loss")
    if not 0.0 < beta < 1e30:
        raise ValueError("beta must be positive")
    if not abs(margin) < 1e30:
        raise ValueError("margin must be finite")
    if rows.sequences < 2 or rows.sequences % 2:
        raise ValueError("preference pairs need an even number of sequences: the chosen ones, then the rejected ones "
                         f"in the same order (got {rows.sequences})")
    if rows.n == 0:
        raise ValueError("preference pairs need rows")
    index, shape, pairs = rows.index, targets.shape, rows.sequences // 2
    ref = None if ref_logps is None else _floats(ref_logps, "ref_logps", shape, index)
    grad, layout = rows.gradient(out, ref) if want_grad else (None, None)
    logps, loss, chosen, rejected = rows.empty(shape), rows.empty(()), rows.empty(pairs), rows.empty(pairs)
    ws, nbytes = rows.workspace()
    spec = N.PreferenceSpec(beta, label_smoothing, margin, mode, 1 if average else 0)
    N.launch("mib_preference_loss", index, rows.spec, spec, _address(ref), loss.data_ptr(), chosen.data_ptr(),
             rejected.data_ptr(), logps.data_ptr(), _address(grad), layout, ws.data_ptr(), nbytes)
    if out is not None:
        increment_version(out)
    return PreferenceLoss(loss, chosen, rejected, logps), grad, ws


def preference_loss(logits, targets, ref_logps=None, *, cu_seqlens=None, beta=0.1, label_smoothing=0.0, margin=0.0,
                    kind="sigmoid", average=False, temperature=1.0, ignore_index=-100):
    """Preference loss over pairs of sequences; returns a ``PreferenceLoss``.

    Of S sequences, sequence i (chosen) is paired with sequence i + S / 2 (rejected).  With ``D`` the sum over a
    sequence's tokens of ``lp - ref_logps`` (their mean with ``average``; no ``ref_logps`` counts as 0) and
    ``h = beta (D_chosen - D_rejected) - margin``, the mean over pairs of ``kind``: "sigmoid"
    ``-(1 - e) log sigmoid(h) - e log sigmoid(-h)`` with ``e = label_smoothing``, "hinge" ``max(0, 1 - h)`` or
    "squared" ``(h - 1/2)^2``.  A sequence without a token counts as D = 0."""
    def evaluate(x):
        return _preference(x, targets, ref_logps, cu_seqlens, beta, label_smoothing, margin, kind, average,
                           temperature, ignore_index, False, None)[::2]
    if logits.requires_grad and torch.is_grad_enabled():
        return PreferenceLoss(*_LossRunc.apply(logits, targets, cu_seqlens, float(temperature), int(ignore_index), evaluate))
    return evaluate(logits)[0]


def preference_loss_grad(logits, targets, ref_logps=None, *, cu_seqlens=None, beta=0.1, label_smoothing=0.0,
                         margin=0.0, kind="sigmoid", average=False, temperature=1.0, ignore_index=-100, out=None):
    """``preference_loss`` and the gradient of its loss over the logits, in their type: ``(PreferenceLoss, grad)``."""
    return _preference(logits, targets, ref_logps, cu_seqlens, beta, label_smoothing, margin, kind, average,
                       temperature, ignore_index, True, out)[:2]
