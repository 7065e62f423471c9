"""The tuning operators together, on crossbar layers: a small language model tuned from preferences and by policy."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _tuner(cuda, noisy=False):
    from memintelli_flash_b200 import lm_tuning
    return lm_tuning.Tuner(lm_tuning.make_engine(cuda, noisy))


def test_preference_tuning_learns_the_rule(cuda):
    t = _tuner(cuda)
    first = t.preference_step()
    assert first["margin"].item() == pytest.approx(0.0, abs=1e-3)          # the model starts as its own reference
    assert first["loss"].item() == pytest.approx(0.6931, abs=1e-3)
    for _ in range(25):
        last = t.preference_step()
    assert last["margin"].item() > 1.0 and last["loss"].item() < 0.35


def test_policy_tuning_step(cuda):
    t = _tuner(cuda, noisy=True)
    before = [p.detach().clone() for p in t.model.parameters()]
    for _ in range(3):
        r = t.policy_step(groups=4, samples=4)
    assert all(torch.isfinite(v).all() for v in r.values())
    assert r["kl"].item() >= 0 and r["norm"].item() > 0
    assert any(not torch.equal(a, b) for a, b in zip(before, t.model.parameters()))


def test_gradients_reach_every_parameter_as_with_torch_operators(cuda):
    """The same loss with torch's embedding, log_softmax and norm: parameter gradients agree to fp32 sums."""
    t = _tuner(cuda)
    ids = t.random_tokens(6, 10)
    from memintelli_flash_b200 import lm_tuning, tuning
    targets = lm_tuning.shifted(ids, 3)
    ref = torch.randn(6, 10, device=cuda)
    tuning.preference_loss(t.model(ids), targets, ref, beta=0.3).loss.backward()
    got = [p.grad.clone() for p in t.model.parameters()]
    norm = tuning.grad_norm(t.model.parameters()).item()
    t.model.zero_grad()
    model = t.model
    model.embed.forward = lambda i: torch.nn.functional.embedding(i, model.embed.weight) * model.embed.scale
    logits = model(ids)
    keep = targets != lm_tuning.IGNORE
    lp = torch.log_softmax(logits, -1).gather(-1, targets.clamp_min(0)[..., None])[..., 0]
    d = torch.where(keep, lp - ref, 0.0).sum(1)
    loss = -torch.nn.functional.logsigmoid(0.3 * (d[:3] - d[3:])).mean()
    loss.backward()
    for a, p in zip(got, model.parameters()):
        assert torch.allclose(a, p.grad, rtol=1e-4, atol=1e-5 * p.grad.abs().max().item())
    want = torch.stack([p.grad.double().square().sum() for p in model.parameters()]).sum().sqrt().item()
    assert norm == pytest.approx(want, rel=1e-4)
