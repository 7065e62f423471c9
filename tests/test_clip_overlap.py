"""Clipping refuses lists in which a tensor that is written shares memory with another.  On the host: the refusal comes
before any device work, so the addresses below are never used."""
import pytest
import torch

from memintelli_flash_b200 import _native as N
from memintelli_flash_b200 import tuning


def clip(ins, outs, numel, in_types=None, out_types=None):
    n = len(ins)
    types = [(N.c_i32 * n)(*(t or [N.F32] * n)) for t in (in_types, out_types)]
    rc = N.lib().mib_clip_grad_norm((N.c_vp * n)(*ins), (N.c_vp * n)(*outs), (N.c_i64 * n)(*numel), *types, n, 2, 1.0, 1e-6,
                                    N.c_vp(0x1000), N.c_vp(0x1000), 0, None)
    assert rc == N.MIB_ERR_PARAM                    # the workspace is too small: what is allowed gets that far
    return b"overlap" in N.lib().mib_last_error()


def test_overlaps_at_the_entry():
    a, b, c = 0x10000, 0x20000, 0x30000
    assert not clip([a, b], [a, b], [10, 10])                               # in place
    assert not clip([a, a + 40], [a, a + 40], [10, 10])                     # neighbours
    assert clip([a, a + 36], [a, a + 36], [10, 10])                         # one element shared
    assert clip([a + 36, c, a], [a + 36, c, a], [10, 5, 10])
    assert clip([a, a], [a, a], [10, 10])                                   # the same twice
    assert clip([a, a + 4], [a, a + 4], [100, 1])                           # one inside the other
    assert not clip([a, a + 4], [a, a + 4], [100, 0])                       # nothing of an empty one
    assert not clip([a, a], [b, c], [10, 10])                               # read twice
    assert clip([a, b], [c, c + 20], [10, 10])                              # written twice
    assert clip([a, b], [b, c], [10, 10])                                   # an output over another's input
    assert clip([a], [a + 4], [10])                                         # over its own, shifted
    assert clip([a], [a], [10], [N.F32], [N.BF16])                          # or as another type
    assert not clip([a], [a + 40], [10], [N.F32], [N.BF16])
    assert not clip([a, a + 20], [b, b + 40], [10, 10], [N.F16, N.F16], [N.F32, N.F32])
    assert clip([a, a + 20], [b, b + 38], [10, 10], [N.F16, N.F16], [N.F32, N.BF16])


@pytest.mark.gpu
def test_overlapping_views_are_refused(cuda):
    base = torch.randn(100, device="cuda")
    kept, other = base.clone(), torch.randn(100, device="cuda")
    for grads, out in (([base[:60], base[50:]], None), ([other, base[:50]], [base, torch.empty(50, device="cuda")]),
                       ([base[:50]], [base[1:51]])):
        with pytest.raises(ValueError, match="overlap"):
            tuning.clip_grad_norm_(grads, 1.0, out=out)
    assert torch.equal(base, kept)
    assert tuning.grad_norm([base[:60], base[50:]]).item() > 0              # reading both is fine
    tuning.clip_grad_norm_([base[:50], base[50:]], 1.0)
    assert not torch.equal(base, kept)
