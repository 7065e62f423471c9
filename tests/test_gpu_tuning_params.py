"""Embedding lookup, its gradient, and gradient-norm clipping against 64-bit restatements.

Tolerances.  A lookup rounds once: one unit in the last place of its type at most half off.  A table row's gradient sums
k tokens in fp32: within (k + 3) 2^-24 times the sum of the terms' magnitudes, then one rounding.  The norm adds at most
64 terms one after another in fp32 and the rest in double: 64 2^-24 relative, 4e-6; a clipped gradient has that, the
coefficient's three roundings, and its own.
"""
import math

import pytest
import torch

from memintelli_flash_b200 import EmbeddingScaled, tuning
from memintelli_flash_b200.NN_layers import embedding_scaled, embedding_scaled_grad

pytestmark = pytest.mark.gpu

ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,hidden", [(1, 1, 1), (1, 50, 1024), (5, 7, 3), (300, 1000, 64), (33, 513, 385),
                                            (2, 100, 4096), (1000, 40, 130), (64, 70000, 20)])
def test_lookup(n, vocab, hidden, dtype, cuda):
    g = gen(n + hidden)
    w = torch.randn(vocab, hidden, generator=g, device="cuda").to(dtype)
    ids = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    assert torch.equal(embedding_scaled(ids, w), w[ids])
    for scale in (hidden ** 0.5, -0.3):
        for i in (ids, ids.int()):
            out = embedding_scaled(i, w, scale)
            want = w[ids].double() * torch.tensor(scale, dtype=torch.float32).double().item()
            assert out.dtype == dtype
            assert bool(((out.double() - want).abs() <= want.abs() * ULP[dtype] + TINY[dtype]).all())


def test_lookup_shapes_strides_and_bad_ids(cuda):
    w = torch.randn(20, 24, device="cuda")
    ids = torch.randint(0, 20, (3, 4, 5), device="cuda")
    assert torch.equal(embedding_scaled(ids, w), w[ids])
    assert torch.equal(embedding_scaled(ids.transpose(0, 2), w), w[ids.transpose(0, 2)])
    assert torch.equal(embedding_scaled(ids, w[:, 1:8]), w[:, 1:8][ids])
    assert torch.equal(embedding_scaled(ids, w[5:15], 1.0)[ids < 10], w[5:15][ids[ids < 10]])
    assert embedding_scaled(ids[:0], w).shape == (0, 4, 5, 24)
    for dtype in DTYPES:
        bad = torch.tensor([0, -1, 20, 2 ** 40, 19], device="cuda")
        out = embedding_scaled(bad, w.to(dtype), 2.0)
        assert torch.isnan(out[1:4]).all() and not torch.isnan(out[[0, 4]]).any()


def grad_oracle(ids, g, vocab, scale, padding=None):
    """(sum, sum of magnitudes, number of terms) per table row, in 64 bits."""
    ids, g = ids.reshape(-1).cpu(), g.reshape(-1, g.shape[-1]).double().cpu()
    keep = (ids >= 0) & (ids < vocab)
    if padding is not None:
        keep &= ids != padding
    z = torch.zeros(vocab, g.shape[1], dtype=torch.float64)
    count = torch.zeros(vocab, dtype=torch.float64).index_add_(0, ids[keep], torch.ones(int(keep.sum()), dtype=torch.float64))
    s = scale if isinstance(scale, int) else torch.tensor(scale, dtype=torch.float32).double().item()
    return z.index_add(0, ids[keep], g[keep]) * s, z.index_add(0, ids[keep], g[keep].abs()) * abs(s), count


def check_grad(out, ids, g, vocab, scale, padding=None, base=None):
    total, mag, count = grad_oracle(ids, g, vocab, scale, padding)
    if base is not None:
        total, mag = total + base.double().cpu(), mag + base.double().cpu().abs()
    tol = (count[:, None] + 3) * 2.0 ** -24 * mag + total.abs() * ULP[out.dtype] + TINY[out.dtype]
    assert bool(((out.double().cpu() - total).abs() <= tol).all())
    none = count == 0
    want = torch.zeros_like(out)[none] if base is None else base[none.to(base.device)]
    assert torch.equal(out[none.to(out.device)], want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,hidden", [(1, 1, 1), (1, 300, 64), (5, 7, 3), (777, 8191, 385), (3000, 11, 40),
                                            (2049, 70000, 16), (5000, 300, 1024), (65, 131, 4100)])
def test_embedding_gradient(n, vocab, hidden, dtype, cuda):
    g = gen(n + vocab)
    ids = (torch.rand(n, generator=g, device="cuda") ** 3 * vocab).long().clamp_max(vocab - 1)
    grad = torch.randn(n, hidden, generator=g, device="cuda").to(dtype)
    out = embedding_scaled_grad(ids, grad, vocab, 0.7)
    assert out.dtype == dtype
    check_grad(out, ids, grad, vocab, 0.7)
    assert torch.equal(out, embedding_scaled_grad(ids.int(), grad, vocab, 0.7))      # the same bits
    wide = torch.full((vocab, hidden), 3.0, device="cuda")
    check_grad(embedding_scaled_grad(ids, grad, vocab, 1.0, out=wide), ids, grad, vocab, 1.0)
    base = torch.randn(vocab, hidden, generator=g, device="cuda")
    acc = embedding_scaled_grad(ids, grad, vocab, 1.5, out=base.clone(), accumulate=True)
    check_grad(acc, ids, grad, vocab, 1.5, base=base)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [2, 31, 64, 65, 500, 20000])
def test_embedding_gradient_of_one_long_run(n, dtype, cuda):
    """Every token the same row, then two rows in turn: runs far longer than any tile."""
    grad = torch.randn(n, 48, generator=gen(n), device="cuda").to(dtype)
    for ids in (torch.full((n,), 5, device="cuda"), torch.arange(n, device="cuda") % 2 * 9):
        check_grad(embedding_scaled_grad(ids, grad, 10, 1.0), ids, grad, 10, 1.0)


def test_embedding_gradient_of_many_tokens(cuda):
    n, vocab = 70001, 151936
    g = gen(1)
    ids = ((vocab + 1.0) ** torch.rand(n, generator=g, device="cuda", dtype=torch.float64)).long() - 1
    ids = torch.randperm(vocab, generator=g, device="cuda")[ids.clamp(0, vocab - 1)]
    grad = torch.randn(n, 8, generator=g, device="cuda")
    check_grad(embedding_scaled_grad(ids, grad, vocab), ids, grad, vocab, 1)


def test_embedding_gradient_padding_strides_and_bad_ids(cuda):
    ids = torch.tensor([[3, 0, 3], [9, -1, 12], [0, 2 ** 33 + 3, 3]], device="cuda")
    grad = torch.randn(3, 3, 50, device="cuda")
    bad = [ids == -1, ids == 12, ids > 100]
    g = grad.clone()
    g[bad[0] | bad[1] | bad[2]] = math.nan            # what does not count is not read into anything
    check_grad(embedding_scaled_grad(ids, g, 12, padding_idx=0), ids, grad, 12, 1, padding=0)
    check_grad(embedding_scaled_grad(ids, g, 12), ids, grad, 12, 1)
    # gradients that are columns of a wider tensor, transposed, or of every other token; a wider table
    check_grad(embedding_scaled_grad(ids, g[..., 3:20], 12), ids, grad[..., 3:20], 12, 1)
    check_grad(embedding_scaled_grad(ids.t(), g.transpose(0, 1), 12), ids.t(), grad.transpose(0, 1), 12, 1)
    flat = torch.randn(10, 8, device="cuda")
    i = torch.randint(0, 4, (5,), device="cuda")
    check_grad(embedding_scaled_grad(i, flat[::2], 4), i, flat[::2], 4, 1)
    table = torch.full((4, 20), 2.0, device="cuda")
    embedding_scaled_grad(i, flat[:5], 4, out=table[:, 5:13])
    check_grad(table[:, 5:13], i, flat[:5], 4, 1)
    assert (table[:, :5] == 2).all() and (table[:, 13:] == 2).all()
    none = torch.full((6,), 7, device="cuda")
    assert not embedding_scaled_grad(none, torch.randn(6, 8, device="cuda"), 9, padding_idx=7).any()
    assert not embedding_scaled_grad(none[:0], torch.randn(0, 8, device="cuda"), 9).any()
    keep = torch.randn(9, 8, device="cuda")
    assert embedding_scaled_grad(none[:0], torch.randn(0, 8, device="cuda"), 9, out=keep, accumulate=True) is keep


def test_embedding_module_and_differences(cuda):
    m = EmbeddingScaled(30, 17, scale=4.0, padding_idx=2, device="cuda")
    assert not m.weight[2].any()
    ids = torch.randint(0, 30, (4, 6), device="cuda")
    ids[0, :3] = 2
    y = torch.randn(4, 6, 17, device="cuda")
    (m(ids) * y).sum().backward()
    check_grad(m.weight.grad, ids, y, 30, 4, padding=2)
    # the loss is linear in the table: a difference of any size gives the slope up to its own rounding, under
    # 4e-6 of the sum of the terms' magnitudes
    d = torch.randn_like(m.weight) / 17
    d[2] = 0
    with torch.no_grad():
        f = lambda w: (embedding_scaled(ids, w, 4.0).double() * y.double()).sum().item()  # noqa: E731
        diff = f(m.weight + d) - f(m.weight - d)
        size = (embedding_scaled(ids, m.weight.abs() + d.abs(), 4.0) * y.abs()).sum().item()
    assert abs(diff / 2 - (m.weight.grad * d).sum().item()) <= 4e-6 * size


def test_tables_past_32_bit_offsets(cuda):
    vocab, hidden = 530000, 4100
    w = torch.zeros(vocab, hidden, dtype=torch.bfloat16, device="cuda")
    w[-3:] = torch.randn(3, hidden, device="cuda").bfloat16()
    ids = torch.tensor([vocab - 1, 0, vocab - 3, vocab - 2, vocab - 1], device="cuda")
    assert torch.equal(embedding_scaled(ids, w), w[ids])
    g = torch.randn(5, hidden, device="cuda").bfloat16()
    out = embedding_scaled_grad(ids, g, vocab, out=w)
    check = torch.stack([g[1], g[2], g[3], (g[0].float() + g[4].float()).bfloat16()])
    assert torch.equal(out[[0, vocab - 3, vocab - 2, vocab - 1]], check)
    assert not out[1:vocab - 3].any()


def test_parameter_operators_in_a_cuda_graph(cuda):
    ids = torch.randint(0, 500, (700,), device="cuda")
    g = torch.randn(700, 96, device="cuda")
    grads = make_grads([5000, 17, 300000], [torch.float32, torch.bfloat16], 2)
    outs = [torch.empty_like(x) for x in grads]
    run = lambda: (embedding_scaled_grad(ids, g, 500), tuning.clip_grad_norm_(grads, 0.5, out=outs))  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = run()
    ids.copy_(torch.randint(0, 500, (700,), device="cuda"))
    graph.replay()
    kept = [x.clone() for x in outs]
    b = run()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and all(torch.equal(x, y) for x, y in zip(kept, outs))


# ---- clipping ------------------------------------------------------------------------------------------
def make_grads(sizes, dtypes, seed, scale=0.05):
    g = gen(seed)
    return [(torch.randn(n, generator=g, device="cuda") * scale).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


def norm_oracle(grads, p):
    flat = torch.cat([g.double().cpu().reshape(-1) for g in grads] + [torch.zeros(1, dtype=torch.float64)]).abs()
    return flat.max().item() if math.isinf(p) else (flat ** p).sum().item() ** (1 / p)


def check_clipped(out, grads, coef):
    for o, g in zip(out, grads):
        want = g.double() * coef
        tol = want.abs() * (ULP[o.dtype] + 4e-6 + 4 * 2.0 ** -24) + TINY[o.dtype]
        assert bool(((o.double() - want).abs() <= tol).all())


LISTS = [[1], [0, 3, 0], [7, 8192, 8193, 1, 100000], [5] * 700 + [300], [1 << 20, 12345], [2] * 1100]


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: f"{len(s)}x{sum(s)}")
def test_clip(sizes, p, cuda):
    for dtypes in ([torch.float32], [torch.bfloat16, torch.float32, torch.float16]):
        grads = make_grads(sizes, dtypes, len(sizes))
        norm = norm_oracle(grads, p)
        assert tuning.grad_norm(grads, p).item() == pytest.approx(norm, rel=5e-6)
        for max_norm in (norm * 0.3, norm * 3):
            coef = min(1.0, max_norm / (norm + 1e-6))
            for out in ([torch.full_like(g, 9) for g in grads], [torch.empty_like(g, dtype=torch.float32) for g in grads]):
                got = tuning.clip_grad_norm_(grads, max_norm, p, out=out)
                assert got.item() == pytest.approx(norm, rel=5e-6) and got.dim() == 0
                check_clipped(out, grads, coef)
            mine = [g.clone() for g in grads]
            tuning.clip_grad_norm_(mine, max_norm, p)
            check_clipped(mine, grads, coef)
            if coef == 1.0:
                assert all(torch.equal(a, b) for a, b in zip(mine, grads))


def test_clip_views_orders_and_parameters(cuda):
    base = torch.randn(5000, device="cuda")
    views = [base[1:1002], base[1003:1010], base[2000:4097].view(-1)]            # off any vector boundary
    want = [v.clone() for v in views]
    rest = base.clone()
    norm = tuning.clip_grad_norm_(views, 1.0).item()
    check_clipped(views, want, 1.0 / (norm_oracle(want, 2) + 1e-6))
    assert norm == pytest.approx(norm_oracle(want, 2), rel=5e-6)
    assert torch.equal(base[:1], rest[:1]) and torch.equal(base[1010:2000], rest[1010:2000]) and torch.equal(base[4097:], rest[4097:])
    # channels-last and transposed gradients; outputs off the inputs' alignment
    a = torch.randn(4, 6, 5, 5, device="cuda").to(memory_format=torch.channels_last)
    b = torch.randn(33, 7, device="cuda").t()
    ref = [a.clone(), b.clone()]
    norm = tuning.clip_grad_norm_([a, b], 0.5).item()
    check_clipped([a, b], ref, 0.5 / (norm + 1e-6))
    buf = torch.empty(1001, device="cuda", dtype=torch.bfloat16)
    src = torch.randn(1000, device="cuda").bfloat16()
    tuning.clip_grad_norm_([src], 2.0, out=[buf[1:]])
    check_clipped([buf[1:]], [src], 2.0 / (norm_oracle([src], 2) + 1e-6))
    m = torch.nn.Linear(30, 20, device="cuda")
    m.weight.grad = torch.randn(20, 30, device="cuda")                          # the bias has none
    w = m.weight.grad.clone()
    assert tuning.grad_norm(m.parameters()).item() == pytest.approx(norm_oracle([w], 2), rel=5e-6)
    tuning.clip_grad_norm_(m.parameters(), 1.0)
    check_clipped([m.weight.grad], [w], 1.0 / (norm_oracle([w], 2) + 1e-6))
    assert tuning.clip_grad_norm_([], 1.0).item() == 0
    assert tuning.clip_grad_norm_([torch.zeros(10, device="cuda")], 1.0).item() == 0


def test_clip_non_finite(cuda):
    for bad, where in ((math.nan, 5), (math.inf, 70000), (-math.inf, 0)):
        for p in (1.0, 2.0, math.inf):
            g = [torch.ones(100000, device="cuda"), torch.ones(7, device="cuda", dtype=torch.bfloat16)]
            g[0][where] = bad
            norm = tuning.clip_grad_norm_(g, 1.0, p).item()
            assert math.isnan(norm) if math.isnan(bad) else norm == math.inf
            want = math.nan if math.isnan(bad) else 0.0                         # 1 / inf; inf * 0 is NaN
            assert torch.equal(g[1].isnan(), torch.full((7,), math.isnan(want), device="cuda"))
            assert g[0][where].isnan()


def test_clip_past_32_bit_offsets(cuda):
    g = torch.zeros((1 << 31) + 1003, dtype=torch.bfloat16, device="cuda")
    g[-5:], g[3] = 3.0, 4.0
    norm = tuning.clip_grad_norm_([g[:7], g[7:]], 0.5).item()
    assert norm == pytest.approx((5 * 9 + 16) ** 0.5, rel=5e-6)
    want = torch.tensor(3.0 * 0.5 / (norm + 1e-6)).bfloat16().item()
    assert g[-5:].tolist() == [want] * 5 and not g[100:-5].any()


def test_clip_same_bits_twice(cuda):
    grads = make_grads([100003, 17, 4096, 250000], [torch.float32, torch.bfloat16], 3)
    outs = [[torch.empty_like(g) for g in grads] for _ in range(2)]
    norms = [tuning.clip_grad_norm_(grads, 0.5, out=o) for o in outs]
    assert torch.equal(norms[0], norms[1]) and all(torch.equal(a, b) for a, b in zip(*outs))


def test_refusals_on_device_tensors(cuda):
    w, ids = torch.randn(9, 8, device="cuda"), torch.zeros(4, dtype=torch.long, device="cuda")
    g = torch.randn(4, 8, device="cuda")
    v = torch.randn(10, 10, device="cuda")
    bad = [
        lambda: embedding_scaled(ids, w.double()),
        lambda: embedding_scaled(ids.float(), w),
        lambda: embedding_scaled(ids.cpu(), w),
        lambda: embedding_scaled(ids, w.t()),
        lambda: embedding_scaled(ids, w[0]),
        lambda: embedding_scaled(ids, w, padding_idx=9),
        lambda: embedding_scaled_grad(ids, g[:3], 9),
        lambda: embedding_scaled_grad(ids, g, 0),
        lambda: embedding_scaled_grad(ids, g, 9, accumulate=True),
        lambda: embedding_scaled_grad(ids, g, 9, out=w[:5]),
        lambda: embedding_scaled_grad(ids, g, 9, out=w.half()),
        lambda: embedding_scaled_grad(ids, g, 9, out=torch.randn(8, 9, device="cuda").t()),
        lambda: embedding_scaled_grad(ids, g, 9, out=torch.randn(1, 8, device="cuda").expand(9, 8)),
        lambda: tuning.clip_grad_norm_([g], -1.0),
        lambda: tuning.clip_grad_norm_([g], math.inf),
        lambda: tuning.clip_grad_norm_([g], 1.0, 3.0),
        lambda: tuning.clip_grad_norm_([g], 1.0, eps=-1.0),
        lambda: tuning.clip_grad_norm_([g.double()], 1.0),
        lambda: tuning.clip_grad_norm_([g, g.cpu()], 1.0),
        lambda: tuning.clip_grad_norm_([v[:, ::2]], 1.0),
        lambda: tuning.clip_grad_norm_([g, g], 1.0),
        lambda: tuning.clip_grad_norm_([g], 1.0, out=[]),
        lambda: tuning.clip_grad_norm_([g], 1.0, out=[g[:3]]),
        lambda: tuning.clip_grad_norm_([v], 1.0, out=[torch.empty(10, 10, device="cuda").t()]),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"refusal {i} did not happen")
