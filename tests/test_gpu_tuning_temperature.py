"""Temperatures far from 1, and those that are refused.

A log-probability is within 1e-5 of the formula's for differences of 64 or less where it counts; here logits / temperature
reach 1e21, and what is allowed beside is two roundings of the result."""
import math

import pytest
import torch

import tuning_oracle as O
from memintelli_flash_b200 import tuning
from test_gpu_tuning_losses import make

pytestmark = pytest.mark.gpu


def test_temperatures(cuda):
    x, t, _ = make(9, 300, torch.float32, 3)
    for temperature in (1e-20, 1e-3, 50.0, 1e20):
        want, _ = O.row_logps(x, t, temperature)
        got = tuning.token_logprobs(x, t, temperature=temperature).double().cpu()
        assert bool(((got - want).abs() <= 1e-5 + want.abs() * 2.0 ** -22).all())
    for temperature in (0.0, -1.0, 1e-40, 1e-31, 1e30, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            tuning.token_logprobs(x, t, temperature=temperature)
