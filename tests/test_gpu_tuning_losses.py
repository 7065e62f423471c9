"""Token log-probabilities, the policy loss and the preference loss against 64-bit restatements.

Tolerances.  Row statistics are fp32: each exponential has a relative error of about 2^-22 plus |arg| 2^-23 with |arg|
under 64 where it counts, a row's sum adds under 64 sequential and 20 tree roundings, so lp is within 1e-5 absolutely,
and the fp32 result adds |lp| 2^-24.  A gradient element c (1{j = t} - p) then is within 3e-5 |c p| of the formula, plus
1e-6 |c| of cancellation at the target, plus one rounding to its type.  Losses are weighted means of functions of lp
with slopes under 4 here: 1e-4 absolutely.
"""
import math

import pytest
import torch

import tuning_oracle as O
from memintelli_flash_b200 import tuning

pytestmark = pytest.mark.gpu

ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
LP_TOL = 1e-5


def make(n, v, dtype, seed, spread=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(n, v, generator=g, device="cuda") * spread).to(dtype)
    t = torch.randint(0, v, (n,), generator=g, device="cuda")
    if n > 3:
        t[::4] = O.IGNORE
    return x, t, g


def near(got, want, tol):
    got, want = got.detach().double().cpu(), want.double().cpu()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ~torch.isnan(want)
    inf = ok & torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    ok &= ~inf
    tol = tol.double()[ok] if isinstance(tol, torch.Tensor) else tol
    assert bool(((got[ok] - want[ok]).abs() <= tol).all()), float(((got[ok] - want[ok]).abs()).max())


def near_logps(got, want):
    near(got, want, LP_TOL + want.abs() * 2.0 ** -23)


def near_grad(got, want, dtype, more=0.0):
    """`want`: the formula's gradient and |c| of each row (tuning_oracle.logit_grad); `more`: relative error of c."""
    want, c = want
    near(got, want, want.abs() * (ULP[dtype] + 3e-5 + more) + 1e-6 * c + TINY[dtype])


SHAPES = [(1, 1), (1, 2), (3, 17), (5, 128), (1, 151936), (37, 1000), (201, 4099), (2, 32003), (700, 33), (9, 70001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v", SHAPES)
def test_logprobs_and_gradient(n, v, dtype, cuda):
    for temperature, idx in ((1.0, torch.int64), (0.7, torch.int32)):
        x, t, g = make(n, v, dtype, n * 31 + v)
        x.requires_grad_(True)
        lp = tuning.token_logprobs(x, t.to(idx), temperature=temperature)
        want, p = O.row_logps(x, t, temperature)
        near_logps(lp, want)
        w = torch.randn(n, generator=g, device="cuda")
        (lp * w).sum().backward()
        near_grad(x.grad, O.logit_grad(p, t, torch.where(t.cpu() == O.IGNORE, 0.0, w.double().cpu()), temperature), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_logprobs_of_strided_logits(dtype, cuda):
    big, _, g = make(6 * 9, 300, dtype, 5)
    big = big.view(6, 9, 300)
    t = torch.randint(0, 200, (6, 9), generator=g, device="cuda")
    # without the last position; columns off a vector boundary; every other row; batch and time swapped
    for view, tt in ((big[:, :-1], t[:, 1:]), (big[..., 3:203], t), (big[::2, 1::2, 7:], t[::2, 1::2]),
                     (big.transpose(0, 1), t.t()), (big.transpose(1, 2)[..., :7], t[:, :1].expand(6, 300) % 7)):
        x = view.detach().requires_grad_(True)
        lp = tuning.token_logprobs(x, tt)
        want, p = O.row_logps(x, tt)
        near_logps(lp, want)
        lp.sum().backward()
        near_grad(x.grad, O.logit_grad(p, tt, torch.ones(tt.shape, dtype=torch.float64)), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [40, 5001])
def test_logprobs_with_masked_columns(dtype, v, cuda):
    lowest = torch.finfo(dtype).min
    x, t, _ = make(12, v, dtype, 3)
    t[:] = torch.arange(12, device="cuda")
    x[1, 5:] = -math.inf                          # most of the row masked
    x[2, 5:] = lowest
    x[3] = -math.inf                              # nothing left: NaN, as the formula
    x[4] = lowest                                 # the lowest value everywhere: uniform
    x[5] = lowest
    x[5, :20] = -math.inf                         # both: uniform over the rest, the target has none
    x[6, 6] = -math.inf                           # the target masked
    x[7, 0] = math.inf                            # NaN
    x[8, v - 1] = math.nan                        # NaN
    x[9] = math.nan
    t[9] = O.IGNORE                               # NaN where the row takes no part
    x[10] = math.inf
    t[10] = O.IGNORE
    t[11] = v                                     # no such column: NaN
    t[1], t[2] = 2, 2
    x.requires_grad_(True)
    lp = tuning.token_logprobs(x, t)
    want, p = O.row_logps(x, t)
    assert want[4].item() == pytest.approx(-math.log(v))
    near_logps(lp, want)
    assert lp[9].item() == 0 and lp[10].item() == 0
    slope = torch.ones(12, dtype=torch.float64)
    slope[9] = slope[10] = 0.0
    lp.sum().backward()
    rows = [0, 1, 2, 4, 5, 6, 9, 10]
    near_grad(x.grad[rows], [a[rows] for a in O.logit_grad(p, t, slope)], dtype)


def policy_inputs(n, v, dtype, seed, cu, per_seq):
    x, t, g = make(n, v, dtype, seed)
    lp, _ = O.row_logps(x, t)
    shift = 0.2 * torch.randn(n, generator=g, device="cuda", dtype=torch.float64).cpu()
    for edge in (0.8, 1.2, 1.3):                  # the slope jumps at the clip bounds: keep tokens off them
        shift = torch.where((shift - math.log(edge)).abs() < 1e-3, shift + 2e-3, shift)
    old = (lp - shift).float().cuda()
    ref = (lp + 0.2 * torch.randn(n, generator=g, device="cuda", dtype=torch.float64).cpu()).float().cuda()
    adv = torch.randn(len(cu) - 1 if per_seq else n, generator=g, device="cuda")
    return x, t, old, adv, ref


def check_policy(r, grad, want, dtype):
    loss, lp, kl, cf, g = want
    near(r.loss, loss, 1e-4)
    near_logps(r.logps, lp)
    near(r.kl, kl, 1e-4)
    near(r.clip_fraction, cf, 1e-5)
    near_grad(grad, g, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["token", "sequence", "sum"])
@pytest.mark.parametrize("n,v,cu", [(1, 64, [0, 1]), (61, 512, [0, 0, 7, 7, 40, 61]), (300, 33, [0, 100, 300]),
                                    (19, 4801, [0, 2, 19])])
def test_policy_loss(n, v, cu, reduction, dtype, cuda):
    x, t, old, adv, ref = policy_inputs(n, v, dtype, n + v, cu, True)
    kw = dict(clip_low=0.2, clip_high=0.3, kl_coef=0.05, reduction=reduction)
    r, grad = tuning.policy_loss_grad(x, t, old, adv, ref, cu_seqlens=torch.tensor(cu, device="cuda"), **kw)
    check_policy(r, grad, O.policy(x, t, old, adv, ref, cu=cu, **kw), dtype)


def test_policy_loss_variants(cuda):
    cu = [3, 30, 30, 50]                          # rows 0-2 and 50-59 belong to no sequence; the second is empty
    x, t, old, adv, ref = policy_inputs(60, 700, torch.float32, 9, cu, True)
    for idx in (torch.int32, torch.int64):
        cul = torch.tensor(cu, device="cuda", dtype=idx)
        for reduction in ("token", "sequence"):
            r, grad = tuning.policy_loss_grad(x, t, old, adv, cu_seqlens=cul, reduction=reduction, temperature=0.8)
            want = O.policy(x, t, old, adv, None, cu=cu, reduction=reduction, temperature=0.8)
            check_policy(r, grad, want, x.dtype)
            assert not grad[:3].any() and not grad[50:].any()
    # advantages per token without sequences, no KL; a (B, T) batch with one advantage per sequence
    x, t, old, adv, ref = policy_inputs(60, 700, torch.float32, 10, cu, False)
    r, grad = tuning.policy_loss_grad(x, t, old, adv, ref)
    check_policy(r, grad, O.policy(x, t, old, adv, ref), x.dtype)
    b = lambda a: a.view(4, 15, *a.shape[1:])  # noqa: E731
    per = adv[:4].contiguous()
    r, grad = tuning.policy_loss_grad(b(x), b(t), b(old), per, b(ref), reduction="sequence", kl_coef=0.1)
    want = O.policy(x, t, old, per, ref, cu=[0, 15, 30, 45, 60], reduction="sequence", kl_coef=0.1)
    check_policy(r._replace(logps=r.logps.view(-1)), grad.view(60, -1), want, x.dtype)


def test_policy_loss_without_tokens(cuda):
    x, t, old, adv, ref = policy_inputs(8, 50, torch.float32, 1, [0, 8], False)
    t[:] = O.IGNORE
    x[3] = math.nan
    for reduction in ("token", "sequence", "sum"):
        cu = torch.tensor([0, 8], device="cuda")
        r, grad = tuning.policy_loss_grad(x, t, old, adv, ref, kl_coef=0.1, reduction=reduction, cu_seqlens=cu)
        assert r.loss.item() == 0 and r.kl.item() == 0 and r.clip_fraction.item() == 0
        assert not r.logps.any() and not grad.any()
    e = torch.empty(0, 50, device="cuda")
    z = torch.empty(0, device="cuda")
    r, grad = tuning.policy_loss_grad(e, z.long(), z, z)
    assert r.loss.item() == 0 and grad.shape == (0, 50)
    assert tuning.token_logprobs(e, z.long()).shape == (0,)


def test_what_stands_at_ignored_rows_is_not_read(cuda):
    cu = [0, 20, 41, 60]
    x, t, old, adv, ref = policy_inputs(60, 700, torch.bfloat16, 12, cu, False)
    cul = torch.tensor(cu, device="cuda")
    a, ga = tuning.policy_loss_grad(x, t, old, adv, ref, kl_coef=0.1, cu_seqlens=cul)
    p, gp = tuning.preference_loss_grad(x[:41], t[:41], ref[:41], cu_seqlens=cul[:3])
    off = t == O.IGNORE
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(torch.float32).max):
        y, u, v, w = x.clone(), old.clone(), adv.clone(), ref.clone()
        y[off], u[off], v[off], w[off] = bad, bad, bad, bad
        b, gb = tuning.policy_loss_grad(y, t, u, v, w, kl_coef=0.1, cu_seqlens=cul)
        q, gq = tuning.preference_loss_grad(y[:41], t[:41], w[:41], cu_seqlens=cul[:3])
        assert all(torch.equal(i, j) for i, j in zip((*a, ga, *p, gp), (*b, gb, *q, gq)))


def test_gradient_against_differences(cuda):
    """Central differences of the loss along random directions of unit length per row.  The loss is good to about
    2e-6, divided by 2h = 0.2; its third derivative along such a direction is under 1, times h^2 / 6 = 1.7e-3: 2e-3."""
    cu = [0, 5, 11, 14, 20]
    x, t, old, adv, ref = policy_inputs(20, 97, torch.float32, 4, cu, True)
    cul = torch.tensor(cu, device="cuda")
    d = torch.randn_like(x)
    d /= d.norm(dim=-1, keepdim=True)
    h = 0.1
    wide = dict(clip_low=0.9, clip_high=4.0, kl_coef=0.1, cu_seqlens=cul, reduction="sequence")
    f = lambda y: tuning.policy_loss(y, t, old, adv, ref, **wide).loss.double().item()  # noqa: E731
    _, grad = tuning.policy_loss_grad(x, t, old, adv, ref, **wide)
    assert abs((f(x + h * d) - f(x - h * d)) / (2 * h) - (grad * d).sum().item()) <= 2e-3
    for kind in ("sigmoid", "squared"):
        kw = dict(cu_seqlens=cul, beta=0.2, kind=kind)
        f = lambda y: tuning.preference_loss(y, t, ref, **kw).loss.double().item()  # noqa: E731
        _, grad = tuning.preference_loss_grad(x, t, ref, **kw)
        assert abs((f(x + h * d) - f(x - h * d)) / (2 * h) - (grad * d).sum().item()) <= 2e-3


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,cu", [(2, 64, [0, 1, 2]), (61, 512, [0, 20, 20, 45, 61]), (1000, 33, [0, 400, 1000]),
                                    (19, 4801, [0, 3, 9, 9, 12, 18, 19])])
def test_preference_loss(n, v, cu, dtype, cuda):
    x, t, _, _, ref = policy_inputs(n, v, dtype, n + 2 * v, cu, True)
    cul = torch.tensor(cu, device="cuda")
    for kw in (dict(), dict(label_smoothing=0.2, margin=0.3, temperature=0.8), dict(kind="hinge", average=True),
               dict(kind="squared", beta=0.5, average=True)):
        for rf in (ref, None):
            if rf is None and not kw.get("average"):
                continue
            r, grad = tuning.preference_loss_grad(x, t, rf, cu_seqlens=cul, **kw)
            loss, chosen, rejected, lp, g = O.preference(x, t, rf, cu, **kw)
            # D sums up to 1000 tokens' lp errors; as they are rounding errors they add to far less than 1000 LP_TOL
            reward_tol = kw.get("beta", 0.1) * LP_TOL * (1 if kw.get("average") else max(b - a for a, b in O.spans(cu)))
            near(r.chosen_rewards, chosen, reward_tol + chosen.abs() * 2.0 ** -23)
            near(r.rejected_rewards, rejected, reward_tol + rejected.abs() * 2.0 ** -23)
            near(r.loss, loss, 4 * reward_tol + loss.abs() * 2.0 ** -22)
            near_logps(r.logps, lp)
            near_grad(grad, g, dtype, 8 * reward_tol)


def test_preference_batch_form_and_untouched_rows(cuda):
    x, t, _, _, ref = policy_inputs(48, 300, torch.float32, 6, [0, 48], True)
    b = lambda a: a.view(4, 12, *a.shape[1:])  # noqa: E731
    r, grad = tuning.preference_loss_grad(b(x), b(t), b(ref))
    loss, _, _, lp, g = O.preference(x, t, ref, [0, 12, 24, 36, 48])
    near(r.loss, loss, 1e-4)
    near_logps(r.logps.view(-1), lp)
    near_grad(grad.view(48, -1), g, x.dtype)
    x[40:] = math.nan                              # rows of no sequence: no part in the loss, zero gradient
    r, grad = tuning.preference_loss_grad(x, t, ref, cu_seqlens=torch.tensor([0, 20, 40], device="cuda"))
    loss, _, _, lp, g = O.preference(x[:40], t[:40], ref[:40], [0, 20, 40])
    near(r.loss, loss, 1e-4)
    near_grad(grad[:40], g, x.dtype)
    assert not grad[40:].any() and not r.logps[40:].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_in_place_gradient_and_views(dtype, cuda):
    cu = [0, 10, 23]
    x, t, old, adv, ref = policy_inputs(23, 1003, dtype, 8, cu, True)
    kw = dict(cu_seqlens=torch.tensor(cu, device="cuda"), kl_coef=0.1)
    r0, g0 = tuning.policy_loss_grad(x, t, old, adv, ref, **kw)
    out = torch.empty(23, 1010, dtype=dtype, device="cuda").fill_(7)[:, 2:1005]
    r1, g1 = tuning.policy_loss_grad(x, t, old, adv, ref, out=out, **kw)
    assert g1 is out and torch.equal(g1, g0) and torch.equal(r0.loss, r1.loss)
    y = x.clone()
    r2, g2 = tuning.policy_loss_grad(y, t, old, adv, ref, out=y, **kw)
    assert g2 is y and torch.equal(g2, g0) and torch.equal(r2.loss, r0.loss)
    p0 = tuning.preference_loss_grad(x, t, ref, cu_seqlens=kw["cu_seqlens"])
    y = x.clone()
    p1 = tuning.preference_loss_grad(y, t, ref, cu_seqlens=kw["cu_seqlens"], out=y)
    assert torch.equal(p0[1], p1[1]) and torch.equal(p0[0].loss, p1[0].loss)


def test_losses_in_autograd(cuda):
    cu = [0, 10, 23]
    x, t, old, adv, ref = policy_inputs(23, 257, torch.float32, 8, cu, True)
    kw = dict(cu_seqlens=torch.tensor(cu, device="cuda"))
    for f, fg, args in ((tuning.policy_loss, tuning.policy_loss_grad, (old, adv, ref)),
                        (tuning.preference_loss, tuning.preference_loss_grad, (ref,))):
        r0, g0 = fg(x, t, *args, **kw)
        y = x.clone().requires_grad_(True)
        r = f(y, t, *args, **kw)
        assert torch.equal(r.loss, r0.loss) and not r.logps.requires_grad
        r.loss.backward(retain_graph=True)
        assert torch.equal(y.grad, g0)
        with pytest.raises(RuntimeError, match="second forward"):
            r.loss.backward()
        y.grad = None
        (f(y, t, *args, **kw).loss * -2.5).backward()
        near(y.grad, g0.double() * -2.5, g0.double().abs().cpu() * 2.5 * 2.0 ** -23)
        with torch.no_grad():
            assert torch.equal(f(y, t, *args, **kw).loss, r0.loss)


def test_same_bits_twice_and_on_another_stream(cuda):
    cu = [0, 100, 333]
    x, t, old, adv, ref = policy_inputs(333, 5003, torch.bfloat16, 8, cu, True)
    kw = dict(cu_seqlens=torch.tensor(cu, device="cuda"))
    a, ga = tuning.policy_loss_grad(x, t, old, adv, ref, **kw)
    p, gp = tuning.preference_loss_grad(x, t, ref, **kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b, gb = tuning.policy_loss_grad(x, t, old, adv, ref, **kw)
        q, gq = tuning.preference_loss_grad(x, t, ref, **kw)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(u, v) for u, v in zip((*a, ga, *p, gp), (*b, gb, *q, gq)))


def test_refusals_on_device_tensors(cuda):
    x, t, old, adv, ref = policy_inputs(8, 50, torch.float32, 1, [0, 8], False)
    cu = torch.tensor([0, 4, 8], device="cuda")
    bad = [
        lambda: tuning.token_logprobs(x.double(), t),
        lambda: tuning.token_logprobs(x, t[:-1]),
        lambda: tuning.token_logprobs(x, t.float()),
        lambda: tuning.token_logprobs(x, t.cpu()),
        lambda: tuning.token_logprobs(x, t, temperature=0.0),
        lambda: tuning.token_logprobs(x[:, :0], t),
        lambda: tuning.policy_loss(x, t, old, adv, clip_low=-0.1),
        lambda: tuning.policy_loss(x, t, old, adv, kl_coef=0.1),
        lambda: tuning.policy_loss(x, t, old, adv, reduction="mean"),
        lambda: tuning.policy_loss(x, t, old, adv, reduction="sequence"),
        lambda: tuning.policy_loss(x, t, old, adv[:3]),
        lambda: tuning.policy_loss(x, t, old[:3], adv),
        lambda: tuning.policy_loss(x, t, old, adv, cu_seqlens=cu.float()),
        lambda: tuning.policy_loss_grad(x, t, old, adv, out=x[:, :-1]),
        lambda: tuning.policy_loss_grad(x, t, old, adv, out=x.half()),
        lambda: tuning.policy_loss_grad(x[:4], t[:4], old[:4], adv[:4], out=x[1:5]),
        lambda: tuning.policy_loss_grad(x, t, old, adv, out=x[:1].expand(8, 50)),
        lambda: tuning.preference_loss(x, t, ref),
        lambda: tuning.preference_loss(x, t, ref, cu_seqlens=torch.tensor([0, 2, 4, 8], device="cuda")),
        lambda: tuning.preference_loss(x, t, ref, cu_seqlens=cu, kind="linear"),
        lambda: tuning.preference_loss(x, t, ref, cu_seqlens=cu, kind="hinge", label_smoothing=0.1),
        lambda: tuning.preference_loss(x, t, ref, cu_seqlens=cu, label_smoothing=0.6),
        lambda: tuning.preference_loss(x, t, ref, cu_seqlens=cu, beta=0.0),
        lambda: tuning.preference_loss(x, t, ref, cu_seqlens=cu, margin=math.inf),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"refusal {i} did not happen")


def test_rising_logits_in_long_rows(cuda):
    """Later parts of a row far above its first ones: the running reference has to follow, by a little or by a lot."""
    for dtype in DTYPES:
        for step in (0.5, 30.0, 200.0, 20000.0):
            x, t, _ = make(200, 40000, dtype, 11, spread=1.0)
            x = (x.float() + (torch.arange(40000, device="cuda") // 5000) * step).to(dtype)
            t[:] = torch.randint(39000, 40000, (200,), device="cuda")
            x[1, :39000] = -math.inf
            x[2, :39000] = torch.finfo(dtype).min
            x[3, 39999], t[3] = math.nan, 5
            want, p = O.row_logps(x, t)
            old = want.nan_to_num(0.0).float().cuda()
            near_logps(tuning.token_logprobs(x, t), want)
            r, grad = tuning.policy_loss_grad(x, t, old, torch.ones(200, device="cuda"), reduction="sum")
            near_logps(r.logps, want)
            rows = [i for i in range(200) if i != 3]
            slope = -torch.exp(want - old.double().cpu())[rows]
            near_grad(grad[rows], O.logit_grad(p[rows], t[rows], slope), dtype, more=2e-5)
            assert grad[3].isnan().all()


def test_rows_past_32_bit_offsets(cuda):
    """More than 2^31 logits: the last rows are where 32-bit offsets would have wrapped."""
    n, v = 16500, 131072
    x = torch.zeros(n, v, dtype=torch.bfloat16, device="cuda")
    rows = torch.tensor([0, 1, n - 2, n - 1], device="cuda")
    x[rows] = (torch.randn(4, v, device="cuda") * 2).bfloat16()
    t = torch.full((n,), O.IGNORE, device="cuda")
    t[rows] = torch.tensor([5, v - 1, 0, v - 1], device="cuda")
    want, p = O.row_logps(x[rows], t[rows])
    near_logps(tuning.token_logprobs(x, t)[rows], want)
    old = torch.zeros(n, device="cuda")
    old[rows] = want.float().cuda()
    r, grad = tuning.policy_loss_grad(x, t, old, torch.ones(n, device="cuda"), reduction="sum", out=x)
    near(r.loss, torch.tensor(-4.0), 1e-4)
    near_grad(grad[rows], O.logit_grad(p, t[rows], -torch.ones(4, dtype=torch.float64)), torch.bfloat16, more=2e-5)


def test_losses_in_a_cuda_graph(cuda):
    cu = [0, 100, 333]
    x, t, old, adv, ref = policy_inputs(333, 5003, torch.bfloat16, 8, cu, True)
    y = policy_inputs(333, 5003, torch.bfloat16, 9, cu, True)[0]
    kw = dict(cu_seqlens=torch.tensor(cu, device="cuda"))
    run = lambda: (tuning.policy_loss_grad(x, t, old, adv, ref, **kw), tuning.preference_loss_grad(x, t, ref, **kw),  # noqa: E731
                   tuning.token_logprobs(x, t))
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (a, ga), (p, gp), lp = run()
    x.copy_(y)
    graph.replay()
    (b, gb), (q, gq), lq = run()
    assert all(torch.equal(u, v) for u, v in zip((*a, ga, *p, gp, lp), (*b, gb, *q, gq, lq)))
