"""The two losses with more behind them: a factor on the loss reaches the gradient before its only rounding.

Tolerances: the gradient's of test_gpu_tuning_losses (statistics and one rounding to the type), for the loss times a factor.
"""
import pytest
import torch

import tuning_oracle as O
from memintelli_flash_b200 import tuning
from test_gpu_tuning_losses import near_grad, policy_inputs

pytestmark = pytest.mark.gpu

N, V, CU = 2000, 1501, [0, 700, 1100, 1500, 2000]


def cases(x, t, old, adv, ref, cu):
    kw = dict(cu_seqlens=torch.tensor(cu, device="cuda"))
    yield (lambda y: tuning.policy_loss(y, t, old, adv, ref, **kw).loss,
           lambda: O.policy(x, t, old, adv, ref, cu=cu)[-1])
    yield (lambda y: tuning.preference_loss(y, t, ref, average=True, **kw).loss,
           lambda: O.preference(x, t, ref, cu, average=True)[-1])


@pytest.mark.parametrize("dtype,factor", [(torch.float16, 65536.0), (torch.bfloat16, -2.5), (torch.float16, 3.0),
                                          (torch.float32, 1e-3)])
def test_a_factor_on_the_loss(dtype, factor, cuda):
    inputs = policy_inputs(N, V, dtype, 3, CU, True)
    for loss, want in cases(*inputs, CU):
        y = inputs[0].clone().requires_grad_(True)
        (loss(y) * factor).backward()
        g, c = want()
        if factor == 65536.0:                      # what the scale is there for: much of it is nothing without it
            assert ((g.abs() < 2.0 ** -25) & (g != 0)).double().mean() > 0.25
        near_grad(y.grad, (g * factor, c * abs(factor)), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v", [(5, 7), (3, 40000), (200, 3001), (1300, 1300), (200, 40001)])
def test_the_same_gradient_with_and_without_autograd(n, v, dtype, cuda):
    """Every form of the row kernels: the gradient of the loss itself has the same bits."""
    cu = [0, n // 2, n]
    x, t, old, adv, ref = policy_inputs(n, v, dtype, 5, cu, True)
    kw = dict(cu_seqlens=torch.tensor(cu, device="cuda"))
    for f, fg, args in ((tuning.policy_loss, tuning.policy_loss_grad, (old, adv, ref)),
                        (tuning.preference_loss, tuning.preference_loss_grad, (ref,))):
        r0, g0 = fg(x, t, *args, **kw)
        y = x.clone().requires_grad_(True)
        r = f(y, t, *args, **kw)
        r.loss.backward()
        assert torch.equal(r.loss, r0.loss) and torch.equal(r.logps, r0.logps) and torch.equal(y.grad, g0)


def test_gradients_of_strided_logits(cuda):
    x, t, old, adv, ref = policy_inputs(60, 130, torch.float32, 5, [0, 60], False)
    b = lambda a: a.view(4, 15, *a.shape[1:])  # noqa: E731
    kw = dict(reduction="sequence", kl_coef=0.1)
    u = torch.where(t < 0, t, t % 97)
    y = x.clone().requires_grad_(True)
    tuning.policy_loss(b(y)[..., 3:100], b(u), b(old), b(adv), b(ref), **kw).loss.backward()
    g = O.policy(x[:, 3:100], u, old, adv, ref, cu=[0, 15, 30, 45, 60], **kw)[-1]
    near_grad(y.grad[:, 3:100], g, x.dtype)
    assert not y.grad[:, :3].any() and not y.grad[:, 100:].any()


def test_the_loss_may_be_changed_in_place(cuda):
    """``loss /= steps``, as in gradient accumulation; the other results too."""
    cu = [0, 10, 23]
    x, t, old, adv, ref = policy_inputs(23, 257, torch.float32, 8, cu, True)
    kw = dict(cu_seqlens=torch.tensor(cu, device="cuda"))
    for f, fg, args in ((tuning.policy_loss, tuning.policy_loss_grad, (old, adv, ref)),
                        (tuning.preference_loss, tuning.preference_loss_grad, (ref,))):
        r0, g0 = fg(x, t, *args, **kw)
        kept = [a.clone() for a in r0]
        y = x.clone().requires_grad_(True)
        r = f(y, t, *args, **kw)
        loss = r.loss
        loss /= 4
        loss.backward()
        assert torch.equal(loss, kept[0] / 4) and all(torch.equal(a, b) for a, b in zip(r[1:], kept[1:]))
        assert torch.equal(y.grad, g0 / 4)
        for a, b in zip((*r[1:], *r0), (*kept[1:], *kept)):
            a *= 0.5
            assert torch.equal(a, b * 0.5)
