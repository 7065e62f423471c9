"""Targets outside the vocabulary.  Tolerances as in test_gpu_tuning_losses."""
import pytest
import torch

import tuning_oracle as O
from memintelli_flash_b200 import tuning
from test_gpu_tuning_losses import make, near_grad, near_logps

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("v", [40, 5001])
def test_gradient_at_a_target_outside_the_vocabulary(v, cuda):
    """The row's log-probability is NaN, and so is its gradient, as the losses' is; without a slope it is zero."""
    x, t, _ = make(6, v, torch.float32, 3)
    t[:] = torch.arange(6, device="cuda")
    t[2], t[4] = v, -7
    x.requires_grad_(True)
    lp = tuning.token_logprobs(x, t)
    want, p = O.row_logps(x, t)
    near_logps(lp, want)
    slope = torch.tensor([1.0, -2.0, 0.5, 1.0, 0.0, 3.0], dtype=torch.float64)
    lp.backward(slope.float().cuda())
    near_grad(x.grad[[0, 1, 3, 4, 5]], [a[[0, 1, 3, 4, 5]] for a in O.logit_grad(p, t, slope)], x.dtype)
    assert x.grad[2].isnan().all()
