"""Layouts of `out`.  Tolerances as in test_gpu_tuning_losses."""
import pytest
import torch

import tuning_oracle as O
from memintelli_flash_b200 import tuning
from test_gpu_tuning_losses import near_grad, policy_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [64, 97, 5003])
def test_out_with_time_and_batch_swapped(v, dtype, cuda):
    """Logits kept as (T, B, V): their (B, T, V) view may take the gradient, in place or beside."""
    B, T = 4, 15
    x, t, old, adv, ref = policy_inputs(B * T, v, dtype, 6, [0, 60], False)
    b = lambda a: a.view(B, T, *a.shape[1:])  # noqa: E731
    r0, g0 = tuning.policy_loss_grad(b(x), b(t), b(old), b(adv), b(ref), kl_coef=0.1)
    p0, q0 = tuning.preference_loss_grad(b(x), b(t), b(ref))
    for pad in (0, 3):
        wide = torch.full((T, B, v + pad), 7.0, dtype=dtype, device="cuda")
        out = wide[..., pad:].transpose(0, 1)
        r, g = tuning.policy_loss_grad(b(x), b(t), b(old), b(adv), b(ref), kl_coef=0.1, out=out)
        assert g is out and torch.equal(g, g0) and torch.equal(r.loss, r0.loss) and bool((wide[..., :pad] == 7).all())
        p, q = tuning.preference_loss_grad(b(x), b(t), b(ref), out=out)
        assert torch.equal(q, q0) and torch.equal(p.loss, p0.loss)
        y = torch.empty_like(wide)[..., pad:].transpose(0, 1).copy_(b(x))
        r1, g1 = tuning.policy_loss_grad(y, b(t), b(old), b(adv), b(ref), kl_coef=0.1)     # a row's sums go by its alignment
        near_grad(g1.view(B * T, v), O.policy(x, t, old, adv, ref, kl_coef=0.1)[-1], dtype)
        r, g = tuning.policy_loss_grad(y, b(t), b(old), b(adv), b(ref), kl_coef=0.1, out=y)
        assert g is y and torch.equal(g, g1) and torch.equal(r.loss, r1.loss)
    rows = torch.empty(T * B * v, dtype=dtype, device="cuda")
    for shape, stride in (((B, T, v), (v - 1, B * v, 1)), ((B, T, v), (v, B * v - 1, 1)), ((B, T, v), (T * v - 1, v, 1))):
        with pytest.raises(ValueError, match="overlap"):
            tuning.policy_loss_grad(b(x), b(t), b(old), b(adv), b(ref), out=rows.as_strided(shape, stride))
