"""``out`` of the losses shares no memory with what else a call reads: a row's gradient may be written before another row's
numbers are read."""
import pytest
import torch

from memintelli_flash_b200 import tuning
from test_gpu_tuning_losses import policy_inputs

pytestmark = pytest.mark.gpu


def test_out_over_other_arguments(cuda):
    n, v, cu = 20, 64, [0, 9, 20]
    x, t, old, adv, ref = policy_inputs(n, v, torch.float32, 4, cu, True)
    buf = torch.zeros(n * v + 40, device="cuda")
    out, cul = buf[:n * v].view(n, v), torch.tensor(cu, device="cuda")
    kept = x.clone()

    def inside(a, at):
        """A copy of ``a`` in the buffer's words from ``at``."""
        words = buf[at:at + a.numel() * a.element_size() // 4]
        return (words if a.dtype == torch.float32 else words.view(a.dtype)).copy_(a)

    def calls(at):
        for k, a in (("targets", t), ("old", old), ("adv", adv), ("ref", ref), ("cu", cul)):
            b = {"targets": t, "old": old, "adv": adv, "ref": ref, "cu": cul, k: inside(a, at)}
            yield lambda: tuning.policy_loss_grad(x, b["targets"], b["old"], b["adv"], b["ref"], cu_seqlens=b["cu"], out=out)
            if k not in ("old", "adv"):
                yield lambda: tuning.preference_loss_grad(x, b["targets"], b["ref"], cu_seqlens=b["cu"], out=out)
    for at in (0, n * v - 2):
        for call in calls(at):
            with pytest.raises(ValueError, match="shares memory"):
                call()
    assert torch.equal(x, kept)
    for call in calls(n * v):                     # behind it in the same buffer
        call()
