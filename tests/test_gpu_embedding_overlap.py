"""``embedding_scaled_grad`` refuses an ``out`` that shares memory with what it reads (``out`` is cleared first)."""
import pytest
import torch

from memintelli_flash_b200.NN_layers import embedding_scaled_grad

pytestmark = pytest.mark.gpu


def test_out_over_the_inputs(cuda):
    buf = torch.randn(40, 8, device="cuda")
    ids = torch.arange(4, device="cuda")
    kept = buf.clone()
    for out, g in ((buf[:9], buf[5:9]), (buf[:9], buf[8:12]), (buf[3:12], buf[:4]), (buf[:4], buf[:4])):
        for accumulate in (False, True):
            with pytest.raises(ValueError, match="shares memory"):
                embedding_scaled_grad(ids, g, out.shape[0], out=out, accumulate=accumulate)
    words = torch.zeros(72, device="cuda")
    with pytest.raises(ValueError, match="shares memory"):
        embedding_scaled_grad(words.view(torch.int64)[8:12], kept[:4], 9, out=words.view(9, 8))
    assert torch.equal(buf, kept)
    out = embedding_scaled_grad(ids, buf[9:13], 9, out=buf[:9])       # side by side
    assert torch.equal(out[:4], kept[9:13]) and not out[4:].any() and torch.equal(buf[9:], kept[9:])
