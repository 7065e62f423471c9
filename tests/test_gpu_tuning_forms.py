"""Every form of the row kernels against 64 bits, with rows that take no part, rows off any vector boundary, and gradients off
the logits' alignment or over them.  Tolerances as in test_gpu_tuning_losses."""
import pytest
import torch

import tuning_oracle as O
from memintelli_flash_b200 import tuning
from test_gpu_tuning_losses import check_policy, make, near_grad, near_logps, policy_inputs

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# a warp per row that reads it twice; a cluster that does; the ring with 128, 256 and 512 threads
FORMS = [(1200, 1201, F32), (1200, 2403, BF16), (2, 170001, F32), (2, 340003, F16), (200, 5003, BF16), (200, 5003, F32),
         (193, 40001, F32), (193, 80009, BF16), (193, 102405, F32)]


def ids(case):
    return "x".join(str(c).replace("torch.", "") for c in case) if isinstance(case, tuple) else None


@pytest.mark.parametrize("case", FORMS, ids=ids)
def test_logprobs(case, cuda):
    n, v, dtype = case
    x, t, g = make(n, v, dtype, n + v)
    if n == 2:
        t[1] = v - 1
    x.requires_grad_(True)
    lp = tuning.token_logprobs(x, t, temperature=0.8)
    want, p = O.row_logps(x, t, 0.8)
    near_logps(lp, want)
    w = torch.randn(n, generator=g, device="cuda")
    (lp * w).sum().backward()
    near_grad(x.grad, O.logit_grad(p, t, torch.where(t.cpu() == O.IGNORE, 0.0, w.double().cpu()), 0.8), dtype)


@pytest.mark.parametrize("case", FORMS, ids=ids)
def test_policy_loss(case, cuda):
    n, v, dtype = case
    cu = [0, 1, n] if n == 2 else [0, n // 5, n // 5, n // 2, n - 3]        # one empty sequence; three rows in none
    x, t, old, adv, ref = policy_inputs(n, v, dtype, n + v, cu, True)
    t[0] = v - 1                                                        # behind the last vector
    lp0, _ = O.row_logps(x[:1], t[:1])
    old[0] = lp0.float().cuda()[0] - 0.05
    x[1] = torch.where(t[1] == O.IGNORE, torch.nan, x[1])               # (row 1 takes part where n is 2)
    ignored = t == O.IGNORE
    y = torch.where(ignored[:, None], torch.zeros_like(x), x)           # the oracle's, without NaN
    kw = dict(clip_low=0.2, clip_high=0.3, reduction="sequence")
    cul = torch.tensor(cu, device="cuda")
    want = O.policy(y, t, old, adv, None, cu=cu, **kw)
    r, grad = tuning.policy_loss_grad(x, t, old, adv, cu_seqlens=cul, **kw)
    check_policy(r, grad, want, dtype)
    wide = torch.full((n, v + 5), 7.0, dtype=dtype, device="cuda")
    for off in (1, 5):                                                  # the gradient's rows off the logits' alignment
        out = wide[:, off:off + v]
        r1, g1 = tuning.policy_loss_grad(x, t, old, adv, cu_seqlens=cul, out=out, **kw)
        assert g1 is out and torch.equal(g1, grad) and all(torch.equal(a, b) for a, b in zip(r1, r))
        assert bool((wide[:, :off] == 7).all()) and bool((wide[:, off + v:] == 7).all())
        wide.fill_(7.0)
    z = x.clone()
    r2, g2 = tuning.policy_loss_grad(z, t, old, adv, cu_seqlens=cul, out=z, **kw)
    assert g2 is z and torch.equal(z, grad) and all(torch.equal(a, b) for a, b in zip(r2, r))


@pytest.mark.parametrize("case", FORMS, ids=ids)
def test_preference_loss(case, cuda):
    n, v, dtype = case
    cu = [0, 1, n] if n == 2 else [0, n // 5, n // 2, n // 2 + 3, n - 3]
    x, t, _, _, ref = policy_inputs(n, v, dtype, n + 2 * v, cu, True)
    t[0] = v - 1
    cul = torch.tensor(cu, device="cuda")
    kw = dict(average=True, label_smoothing=0.1)
    want = O.preference(x, t, ref, cu, **kw)
    r, grad = tuning.preference_loss_grad(x, t, ref, cu_seqlens=cul, **kw)
    near_logps(r.logps, want[3])
    near_grad(grad, want[4], dtype, 1e-5)
    wide = torch.full((n, v + 3), 7.0, dtype=dtype, device="cuda")
    tuning.preference_loss_grad(x, t, ref, cu_seqlens=cul, out=wide[:, 3:], **kw)
    near_grad(wide[:, 3:], want[4], dtype, 1e-5)
    assert bool((wide[:, :3] == 7).all())
    z = x.clone()
    tuning.preference_loss_grad(z, t, ref, cu_seqlens=cul, out=z, **kw)
    assert torch.equal(z, grad)


def test_ignored_rows_past_32_bit_offsets(cuda):
    n, v = 16500, 131072
    x = torch.randn(1, v, device="cuda").bfloat16().expand(n, v).contiguous()
    t = torch.full((n,), O.IGNORE, device="cuda")
    t[5] = 3
    one = torch.ones(n, device="cuda")
    _, grad = tuning.policy_loss_grad(x, t, -10 * one, one, reduction="sum", out=x)
    assert grad[5].any()
    grad[5] = 0
    assert not any(bool(g.any()) for g in grad.split(2000))
