"""What an operator writes into a caller's tensor counts as an in-place change: a graph that saved it refuses to go on."""
import pytest
import torch

from memintelli_flash_b200 import tuning
from memintelli_flash_b200.NN_layers import embedding_scaled_grad
from test_gpu_tuning_losses import policy_inputs

pytestmark = pytest.mark.gpu


def test_logits_overwritten_by_their_gradient(cuda):
    cu = torch.tensor([0, 4, 8], device="cuda")
    x, t, old, adv, ref = policy_inputs(8, 50, torch.float32, 1, [0, 8], False)
    for write in (lambda z: tuning.policy_loss_grad(z, t, old, adv, ref, out=z),
                  lambda z: tuning.preference_loss_grad(z, t, ref, cu_seqlens=cu, out=z)):
        y = x.clone().requires_grad_(True)
        z = y * 1.0
        lp = tuning.token_logprobs(z, t)
        with torch.no_grad():
            write(z)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            lp.sum().backward()


def test_versions_go_up(cuda):
    cu = torch.tensor([0, 4, 8], device="cuda")
    x, t, old, adv, ref = policy_inputs(8, 50, torch.float32, 1, [0, 8], False)
    ids, g = torch.arange(4, device="cuda"), torch.randn(4, 8, device="cuda")
    out, table, more, none = torch.empty_like(x), torch.zeros(9, 8, device="cuda"), torch.empty_like(g), torch.empty(0, 50, device="cuda")

    def moves(a, f):
        before = a._version
        f()
        return a._version > before
    assert moves(out, lambda: tuning.policy_loss_grad(x, t, old, adv, ref, out=out))
    assert moves(out, lambda: tuning.preference_loss_grad(x, t, ref, cu_seqlens=cu, out=out))
    assert moves(table, lambda: embedding_scaled_grad(ids, g, 9, out=table))
    assert moves(table, lambda: embedding_scaled_grad(ids, g, 9, out=table, accumulate=True))
    assert moves(more, lambda: tuning.clip_grad_norm_([g], 1.0, out=[more]))
    assert moves(g, lambda: tuning.clip_grad_norm_([g, more], 1.0)) and moves(more, lambda: tuning.clip_grad_norm_(iter([g, more]), 1.0))
    assert not moves(g, lambda: tuning.clip_grad_norm_([g], 1.0, out=[more]))
    assert not moves(g, lambda: tuning.grad_norm([g])) and not moves(x, lambda: tuning.policy_loss_grad(x, t, old, adv, ref))
    w = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    w.grad = torch.ones(3, device="cuda")
    assert moves(w.grad, lambda: tuning.clip_grad_norm_([w], 1.0)) and w._version == 0
    with torch.inference_mode():                   # tensors without a version
        a = torch.ones(5, device="cuda")
        tuning.clip_grad_norm_([a], 1.0)
        assert a[0].item() == pytest.approx(5 ** -0.5, rel=1e-5)
