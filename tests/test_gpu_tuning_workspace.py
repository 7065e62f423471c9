"""The losses make nothing of what their workspace held before."""
import pytest
import torch

from memintelli_flash_b200 import tuning
from memintelli_flash_b200.tuning import losses
from test_gpu_tuning_losses import policy_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,v", [(8, 50), (300, 700), (1300, 1300), (200, 5003), (200, 40001), (3, 40001)])
def test_workspaces_of_any_content(n, v, cuda, monkeypatch):
    cu = [0, n // 4, n // 2, n // 2, n]
    x, t, old, adv, ref = policy_inputs(n, v, torch.bfloat16, 7, cu, True)
    kw = dict(cu_seqlens=torch.tensor(cu, device="cuda"))

    def run():
        y = x.clone().requires_grad_(True)
        r = tuning.policy_loss(y, t, old, adv, ref, reduction="sequence", **kw)
        p = tuning.preference_loss(y, t, ref, **kw)
        (r.loss + p.loss).backward()
        a, ga = tuning.policy_loss_grad(x, t, old, adv, ref, **kw)
        b, gb = tuning.preference_loss_grad(x, t, ref, **kw)
        return [*r, *p, y.grad, *a, ga, *b, gb]
    plain, want = losses._Rows.workspace, run()
    assert all(torch.isfinite(a).all() for a in want)
    for byte in (0, 1, 0x7f, 0xff):
        def filled(self):
            ws, n = plain(self)
            return ws.fill_(byte), n
        monkeypatch.setattr(losses._Rows, "workspace", filled)
        assert all(torch.equal(a, b) for a, b in zip(run(), want))
