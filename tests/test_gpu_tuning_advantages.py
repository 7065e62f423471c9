"""Which advantage a row of packed sequences gets.  Tolerances as in test_gpu_tuning_losses."""
import pytest
import torch

import tuning_oracle as O
from memintelli_flash_b200 import tuning
from test_gpu_tuning_losses import check_policy, policy_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cu", [[0, 2, 2, 3], [0, 0, 3, 3], [0, 1, 2, 3]])
def test_as_many_sequences_as_rows(cu, cuda):
    """With offsets, one advantage per sequence, also where there are as many sequences as rows."""
    x, t, old, adv, ref = policy_inputs(3, 97, torch.float32, 2, cu, True)
    cul = torch.tensor(cu, device="cuda")
    of_row = torch.stack([adv[i] for i, (a, b) in enumerate(O.spans(cu)) for _ in range(a, b)])
    for reduction in ("token", "sequence", "sum"):
        kw = dict(clip_low=0.2, clip_high=0.3, kl_coef=0.05, reduction=reduction)
        r, grad = tuning.policy_loss_grad(x, t, old, adv, ref, cu_seqlens=cul, **kw)
        check_policy(r, grad, O.policy(x, t, old, of_row, ref, cu=cu, **kw), x.dtype)
        for per, a in (("sequence", of_row), ("token", adv)):
            r, grad = tuning.policy_loss_grad(x, t, old, adv, ref, cu_seqlens=cul, advantages_per=per, **kw)
            check_policy(r, grad, O.policy(x, t, old, a, ref, cu=cu, **kw), x.dtype)
            assert torch.equal(tuning.policy_loss(x, t, old, adv, ref, cu_seqlens=cul, advantages_per=per, **kw).loss, r.loss)


def test_refusals(cuda):
    cu = [0, 2, 8]
    x, t, old, adv, ref = policy_inputs(8, 50, torch.float32, 1, cu, False)
    cul = torch.tensor(cu, device="cuda")
    for bad in (lambda: tuning.policy_loss(x, t, old, adv, cu_seqlens=cul, advantages_per="sequence"),
                lambda: tuning.policy_loss(x, t, old, adv[:2], cu_seqlens=cul, advantages_per="token"),
                lambda: tuning.policy_loss(x, t, old, adv, advantages_per="sequence"),
                lambda: tuning.policy_loss(x, t, old, adv, advantages_per="row")):
        with pytest.raises(ValueError):
            bad()
