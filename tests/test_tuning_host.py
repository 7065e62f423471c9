"""Host-side checks of the tuning operators: refusals before any device work, workspaces, and CPU tensors."""
import ctypes

import pytest
import torch

from memintelli_flash_b200 import _native as N
from memintelli_flash_b200 import tuning
from memintelli_flash_b200.NN_layers import embedding_scaled, embedding_scaled_grad

FAKE = ctypes.c_void_p(0x1000)          # never dereferenced: every call below fails its host checks


def _rows(**kw):
    f = dict(logits=0x1000, targets=0x1000, cu_seqlens=None, rows=4, cols=8, layout=N.OutLayout(4, 0, 8, 1),
             ignore_index=-100, sequences=0, rows_per_sequence=0, temperature=1.0, dtype=N.F32, targets_i64=1, cu_i64=1,
             reserved=0)
    f.update(kw)
    return N.TokenRows(**f)


def test_cpu_tensors_are_refused():
    x, t = torch.randn(4, 8), torch.zeros(4, dtype=torch.long)
    for f in (lambda: tuning.token_logprobs(x, t), lambda: tuning.policy_loss(x, t, x[:, 0], x[:, 0]),
              lambda: tuning.preference_loss(x, t), lambda: tuning.clip_grad_norm_([x], 1.0),
              lambda: tuning.grad_norm([x]), lambda: embedding_scaled(t, x), lambda: embedding_scaled_grad(t, x, 5)):
        with pytest.raises(ValueError, match="CUDA"):
            f()


def test_token_rows_are_checked():
    L = N.lib()
    lp = lambda r: L.mib_token_logps(r, FAKE, None, None)  # noqa: E731
    assert lp(_rows(logits=None)) == N.MIB_ERR_PARAM
    assert lp(_rows(targets=None)) == N.MIB_ERR_PARAM
    assert lp(_rows(logits=0x1002)) == N.MIB_ERR_PARAM                       # fp32 off its alignment
    assert lp(_rows(targets=0x1004)) == N.MIB_ERR_PARAM                      # int64 off its alignment
    assert lp(_rows(dtype=3)) == N.MIB_ERR_UNSUPPORTED
    assert lp(_rows(rows=0)) == N.MIB_ERR_SHAPE
    assert lp(_rows(cols=0)) == N.MIB_ERR_SHAPE
    assert lp(_rows(temperature=0.0)) == N.MIB_ERR_PARAM
    assert lp(_rows(temperature=float("nan"))) == N.MIB_ERR_PARAM
    assert lp(_rows(layout=N.OutLayout(4, 0, 7, 1))) == N.MIB_ERR_SHAPE      # rows overlap
    assert lp(_rows(layout=N.OutLayout(4, 0, 8, 2))) == N.MIB_ERR_SHAPE
    assert L.mib_token_logps(_rows(), None, None, None) == N.MIB_ERR_PARAM
    assert L.mib_token_logps(_rows(), FAKE, ctypes.c_void_p(0x1008), None) == N.MIB_ERR_PARAM    # statistics off 16 bytes
    assert L.mib_token_logps_grad(_rows(), None, FAKE, FAKE, N.OutLayout(4, 0, 8, 1), None) == N.MIB_ERR_PARAM


def test_loss_arguments_are_checked():
    L = N.lib()
    lay = N.OutLayout(4, 0, 8, 1)

    def policy(rows=None, **kw):
        s = dict(clip_low=0.2, clip_high=0.2, kl_coef=0.0, reduction=0, adv_per_sequence=0)
        s.update(kw)
        return L.mib_policy_loss(rows or _rows(), N.PolicySpec(**s), FAKE, FAKE, None, FAKE, FAKE, FAKE, lay, FAKE, 16,
                                 None)
    assert policy(clip_low=-0.1) == N.MIB_ERR_PARAM
    assert policy(clip_low=1.1) == N.MIB_ERR_PARAM
    assert policy(kl_coef=0.1) == N.MIB_ERR_PARAM                            # no reference
    assert policy(reduction=3) == N.MIB_ERR_PARAM
    assert policy(reduction=1) == N.MIB_ERR_PARAM                            # no sequences
    assert policy(adv_per_sequence=1) == N.MIB_ERR_PARAM
    assert policy(_rows(sequences=2)) == N.MIB_ERR_PARAM                     # neither offsets nor a length
    assert policy() == N.MIB_ERR_PARAM and b"workspace" in L.mib_last_error()

    def preference(rows=None, **kw):
        s = dict(beta=0.1, label_smoothing=0.0, margin=0.0, kind=0, average=0)
        s.update(kw)
        return L.mib_preference_loss(rows or _rows(sequences=2, rows_per_sequence=2), N.PreferenceSpec(**s), None, FAKE,
                                     FAKE, FAKE, FAKE, FAKE, lay, FAKE, 16, None)
    assert preference(_rows()) == N.MIB_ERR_SHAPE
    assert preference(_rows(sequences=3, rows_per_sequence=1)) == N.MIB_ERR_SHAPE
    assert preference(beta=0.0) == N.MIB_ERR_PARAM
    assert preference(kind=3) == N.MIB_ERR_PARAM
    assert preference(kind=1, label_smoothing=0.1) == N.MIB_ERR_PARAM
    assert preference(label_smoothing=0.7) == N.MIB_ERR_PARAM
    assert preference(margin=float("inf")) == N.MIB_ERR_PARAM
    assert preference() == N.MIB_ERR_PARAM and b"workspace" in L.mib_last_error()


def test_embedding_arguments_are_checked():
    L = N.lib()
    assert L.mib_embedding_lookup(None, 1, 4, FAKE, N.F32, 9, 8, 8, 1.0, FAKE, None) == N.MIB_ERR_PARAM
    assert L.mib_embedding_lookup(FAKE, 1, 4, FAKE, 7, 9, 8, 8, 1.0, FAKE, None) == N.MIB_ERR_UNSUPPORTED
    assert L.mib_embedding_lookup(FAKE, 1, 4, FAKE, N.F32, 9, 8, 7, 1.0, FAKE, None) == N.MIB_ERR_SHAPE
    assert L.mib_embedding_lookup(FAKE, 1, 0, FAKE, N.F32, 9, 8, 8, 1.0, FAKE, None) == N.MIB_ERR_SHAPE
    g = lambda gt=N.F32, ot=N.F32, ld=8, ws=16: L.mib_embedding_grad(  # noqa: E731
        FAKE, 1, 4, FAKE, gt, 8, 9, 8, 1.0, -1, FAKE, ot, ld, 0, FAKE, ws, None)
    assert g(gt=N.F32, ot=N.BF16) == N.MIB_ERR_UNSUPPORTED
    assert g(gt=N.BF16, ot=N.F16) == N.MIB_ERR_UNSUPPORTED
    assert g(ld=7) == N.MIB_ERR_SHAPE
    assert g() == N.MIB_ERR_PARAM and b"workspace" in L.mib_last_error()
    odd = ctypes.c_void_p(0x1002)
    assert L.mib_embedding_lookup(FAKE, 1, 4, odd, N.F32, 9, 8, 8, 1.0, FAKE, None) == N.MIB_ERR_PARAM
    assert L.mib_embedding_lookup(odd, 0, 4, FAKE, N.F32, 9, 8, 8, 1.0, FAKE, None) == N.MIB_ERR_PARAM
    n = N.c_i64(0)
    assert L.mib_embedding_grad_workspace(0, 9, 8, n) == N.MIB_ERR_SHAPE
    assert L.mib_embedding_grad_workspace(16384, 151936, 1024, n) == 0 and n.value > 8 * 16384


def test_clip_arguments_are_checked():
    L = N.lib()
    ptrs, numel, types = (N.c_vp * 1)(0x1000), (N.c_i64 * 1)(4), (N.c_i32 * 1)(N.F32)
    n = N.c_i64(0)
    assert L.mib_clip_grad_norm_workspace(1, n) == 0 and n.value > 0
    call = lambda norm_type=2, max_norm=1.0, ws=0, types=types, numel=numel, norm=FAKE: L.mib_clip_grad_norm(  # noqa: E731
        ptrs, ptrs, numel, types, types, 1, norm_type, max_norm, 1e-6, norm, FAKE, ws, None)
    assert call(norm_type=3) == N.MIB_ERR_UNSUPPORTED
    assert call(max_norm=-1.0) == N.MIB_ERR_PARAM
    assert call(types=(N.c_i32 * 1)(5)) == N.MIB_ERR_UNSUPPORTED
    assert call(numel=(N.c_i64 * 1)(-1)) == N.MIB_ERR_SHAPE
    assert call(norm=None) == N.MIB_ERR_PARAM
    assert call() == N.MIB_ERR_PARAM and b"workspace" in L.mib_last_error()


def test_an_empty_list_has_norm_zero():
    assert tuning.grad_norm([]).item() == 0
    assert tuning.clip_grad_norm_(iter(()), 1.0).item() == 0
