"""Sums of log-probabilities over long sequences against 64 bits.

Tolerance.  A row's log-probability is off by the roundings of its exponentials and of the sums that join them.  Those are
independent from row to row and as often up as down; the last joins weigh most, each within 2^-24 of the sum, so that the
whole is under 5e-8 (root mean square) a row.  Over n rows that adds up to 5e-8 sqrt(n), and five times that is allowed.
An error with a mean would grow with n instead: 1e-8 a row is 8e-5 over 8000 rows, where 2.2e-5 are allowed.
"""
import math

import pytest
import torch

from memintelli_flash_b200 import tuning

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ROWS = 8000
TOL = 5 * 5e-8 * math.sqrt(ROWS)


def logps64(x, t, temperature):
    out = []
    for i in range(0, x.shape[0], 1000):
        y = x[i:i + 1000].double() / temperature
        out.append(y.gather(1, t[i:i + 1000, None])[:, 0] - torch.logsumexp(y, 1))
    return torch.cat(out)


def rows(vocab, dtype, spread, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(2 * ROWS, vocab, generator=g, device="cuda").mul_(spread)
    x += 3.0 * torch.randn(2 * ROWS, 1, generator=g, device="cuda")
    return x.to(dtype), torch.randint(0, vocab, (2 * ROWS,), generator=g, device="cuda")


def rewards(x, t, ref, temperature):
    cu = torch.tensor([0, ROWS, 2 * ROWS], device="cuda")
    r = tuning.preference_loss(x, t, ref, cu_seqlens=cu, beta=1.0, temperature=temperature)
    return torch.cat([r.chosen_rewards, r.rejected_rewards]).double()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [128, 500, 2000, 8000, 32003])
def test_summed_log_ratios_have_no_mean_error(vocab, dtype, cuda):
    off = {}
    for temperature in (1.0, 0.7):
        for spread in (0.05, 1.0, 5.0):
            x, t = rows(vocab, dtype, spread, vocab)
            lp = logps64(x, t, temperature)
            ref = lp.float()                           # the sequences' exact log ratio is this rounding's alone
            want = (lp - ref.double()).view(2, ROWS).sum(1)
            got = rewards(x, t, ref, temperature)
            off[temperature, spread] = float((got - want).abs().max())
    assert max(off.values()) <= TOL, off


@pytest.mark.parametrize("dtype", DTYPES)
def test_log_ratio_of_a_policy_to_itself_has_no_mean(dtype, cuda):
    """``token_logprobs`` against the losses' own log-probabilities: their difference is the former's last rounding, which
    is even over one unit in the last place: a root mean square of 1 / sqrt(12) of it."""
    for temperature in (1.0, 0.7):
        x, t = rows(3001, dtype, 2.5, 7)
        old = tuning.token_logprobs(x, t, temperature=temperature)
        unit = torch.exp2(torch.floor(torch.log2(old.double().abs())) - 23)
        tol = TOL + 5 * (unit.square().view(2, ROWS).sum(1) / 12).sqrt()
        assert bool((rewards(x, t, old, temperature).abs() <= tol).all())
