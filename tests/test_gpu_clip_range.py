"""Norms and clipping of gradients far from 1.  Tolerances as in test_gpu_tuning_params."""
import math

import pytest
import torch

from memintelli_flash_b200 import tuning
from test_gpu_tuning_params import check_clipped, norm_oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-30, 1e-22, 1e-3, 1e15, 1e21, 1e30])
def test_norm_of_small_and_large_gradients(size, dtype, cuda):
    """The squares of fp32 and bf16 gradients pass fp32's range on both sides."""
    g = [(torch.randn(n, device="cuda") * size).to(dtype) for n in (70001, 3, 9000)]
    g[1][1] = 0
    for p in (1.0, 2.0, math.inf):
        assert tuning.grad_norm(g, p).item() == pytest.approx(norm_oracle(g, p), rel=5e-6)
    norm = norm_oracle(g, 2)
    out = [torch.empty_like(x) for x in g]
    tuning.clip_grad_norm_(g, size, out=out, eps=0.0)
    check_clipped(out, g, min(1.0, size / norm))
