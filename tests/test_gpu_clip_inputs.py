"""What gradient clipping takes as gradients.  Tolerances as in test_gpu_tuning_params."""
import pytest
import torch

from memintelli_flash_b200 import tuning
from test_gpu_tuning_params import check_clipped, norm_oracle

pytestmark = pytest.mark.gpu


def test_leaf_tensors_are_parameters(cuda):
    """As torch's function: a leaf that requires a gradient stands for its gradient and is never scaled itself."""
    a = torch.randn(300, device="cuda", requires_grad=True)
    b = torch.randn(7, 5, device="cuda", requires_grad=True)
    (a.sum() * 3 + (b * b).sum()).backward()
    none = torch.randn(4, device="cuda", requires_grad=True)          # has no gradient: skipped
    kept, want = [a.detach().clone(), b.detach().clone(), none.detach().clone()], [a.grad.clone(), b.grad.clone()]
    assert tuning.grad_norm([a, none, b]).item() == pytest.approx(norm_oracle(want, 2), rel=5e-6)
    norm = tuning.clip_grad_norm_([a, none, b], 0.5).item()
    assert norm == pytest.approx(norm_oracle(want, 2), rel=5e-6)
    check_clipped([a.grad, b.grad], want, 0.5 / (norm + 1e-6))
    assert all(torch.equal(x, k) for x, k in zip((a, b, none), kept))
    # a gradient that is itself part of a graph is a gradient
    g, = torch.autograd.grad((b ** 3).sum(), b, create_graph=True)
    assert g.requires_grad and tuning.grad_norm([g]).item() == pytest.approx(norm_oracle([g.detach()], 2), rel=5e-6)
