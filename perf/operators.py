"""Measured cases of the language-model tuning operators: scaled embedding lookup and its gradient, token
log-probabilities, the clipped policy loss and the paired preference loss with their logit gradients, and the global
gradient norm with clipping.

``run(state)`` makes one pass.  With ``own`` false it evaluates the formula in elementary torch operations in 32 bits,
rounded once at the end; with ``own`` true it makes the call a user of the package makes.  ``exact`` restates the
definitions in 64 bits.

Formulas (rows r of a (N, V) logit block, target t_r, temperature T, x = logits / T):

    lp_r = x[r, t_r] - log sum_j exp(x[r, j])
    policy:     ratio = exp(lp - old), loss = sum_r w_r (-min(ratio A, clamp(ratio, 1 - cl, 1 + ch) A)
                                                       + b (exp(ref - lp) - (ref - lp) - 1))
    preference: D_s = sum over sequence s of (lp - ref), h = beta (D_chosen - D_rejected),
                loss = mean over pairs of -(1 - eps) log sigmoid(h) - eps log sigmoid(-h)
    embedding:  out_i = scale W[ids_i], dW[v] = scale sum over i with ids_i = v of dout_i
    clipping:   n = sqrt(sum of all g^2), g <- g min(1, max_norm / (n + 1e-6))
"""
import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
IGNORE = -100
# decoder geometry of this package's prefill driver (Qwen3Arch) and its 8 x 2048-token benchmark
VOCAB, HIDDEN, LAYERS, INTER, Q_DIM, KV_DIM, HEAD_DIM = 151936, 1024, 28, 3072, 2048, 1024, 128


def listed():
    return [
        # one token of one sequence: the lookup in front of a decoding step, all latency
        dict(name="lookup_one_token", op="lookup", n=1, vocab=VOCAB, hidden=HIDDEN, dtype="bf16", scale=32.0),
        # the 8 x 2048-token batch of the prefill driver, its fp32 table
        dict(name="lookup_batch", op="lookup", n=16384, vocab=VOCAB, hidden=HIDDEN, dtype="fp32", scale=1.0),
        # a small fine-tuning batch, odd vocabulary and width (rows off any vector boundary)
        dict(name="embed_grad_odd", op="embed_grad", n=777, vocab=8191, hidden=385, dtype="fp16", scale=19.6,
             accumulate=False),
        # the full training batch: dense fp32 gradient of the whole table
        dict(name="embed_grad_batch", op="embed_grad", n=16384, vocab=VOCAB, hidden=HIDDEN, dtype="fp32", scale=1.0,
             accumulate=False),
        # scoring one sampled token against the crossbar lm_head's fp32 logits: one row, all latency
        dict(name="logps_one_token", op="logps", n=1, vocab=VOCAB, seqs=1, dtype="fp32", temperature=1.0),
        # scoring a batch of answers under the reference model, at the sampling temperature
        dict(name="logps_batch", op="logps", n=2048, vocab=VOCAB, seqs=8, dtype="bf16", temperature=0.7),
        # toy policy step of a small test model: a few launches' worth of latency
        dict(name="policy_small", op="policy", n=96, vocab=512, seqs=2, dtype="fp32", kl_coef=0.0,
             reduction="token", temperature=1.0),
        # a policy-gradient micro-batch on the crossbar lm_head's fp32 logits, sequence-wise mean, KL to a reference
        dict(name="policy_fp32", op="policy", n=2047, vocab=VOCAB, seqs=8, dtype="fp32", kl_coef=0.05,
             reduction="sequence", temperature=1.0),
        # four preference pairs of ragged answers, odd vocabulary: rows start on every alignment
        dict(name="preference_odd", op="preference", n=1501, vocab=32003, seqs=8, dtype="bf16", smoothing=0.1,
             temperature=1.0),
        # eight pairs on the full vocabulary
        dict(name="preference_batch", op="preference", n=2048, vocab=VOCAB, seqs=16, dtype="bf16", smoothing=0.0,
             temperature=1.0),
        # every parameter of a three-layer perceptron, 784-512-128-10 (the package's example workload)
        dict(name="clip_mlp", op="clip", layout="mlp", tensors=6, elements=784 * 512 + 512 * 128 + 128 * 10 + 650,
             dtype="fp32"),
        # every parameter of the prefill driver's decoder, fp32 gradients: 3 GB in 311 tensors
        dict(name="clip_decoder", op="clip", layout="decoder", tensors=3 + 11 * LAYERS, elements=751632384,
             dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["lookup", "embed_grad", "logps", "policy", "preference", "clip"])
    dtype = rng.choice(sorted(DTYPES))
    if op in ("lookup", "embed_grad"):
        vocab, hidden = _log_int(rng, 128, VOCAB), _log_int(rng, 64, 4096)
        hidden = min(hidden, VOCAB * HIDDEN // vocab)
        if rng.random() < 0.6:
            hidden = max(64, hidden // 64 * 64)
        n = min(_log_int(rng, 1, 65536), max(1, 16384 * HIDDEN // hidden))
        case = dict(op=op, n=n, vocab=vocab, hidden=hidden, dtype=dtype, scale=rng.choice([1.0, round(hidden ** 0.5, 3)]))
        if op == "embed_grad":
            case["accumulate"] = rng.random() < 0.4
        return case
    if op in ("logps", "policy", "preference"):
        vocab = _log_int(rng, 128, VOCAB)
        if rng.random() < 0.5:
            vocab = max(128, vocab // 64 * 64)
        seqs = 1 if op == "logps" else 2 * _log_int(rng, 1, 16)
        n = min(_log_int(rng, seqs, 16384), max(seqs, 2047 * VOCAB // vocab))
        case = dict(op=op, n=n, vocab=vocab, seqs=seqs, dtype=dtype, temperature=rng.choice([1.0, 1.0, 0.7]))
        if op == "policy":
            case.update(kl_coef=rng.choice([0.0, 0.05]), reduction=rng.choice(["token", "sequence"]))
        elif op == "preference":
            case.update(smoothing=rng.choice([0.0, 0.1]))
        return case
    return dict(op="clip", layout="random", tensors=_log_int(rng, 1, 400), elements=_log_int(rng, 1000, 600_000_000),
                dtype=dtype)


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _token_ids(n, vocab, g):
    """Token ids by Zipf's law, p(rank k) = log((k + 2) / (k + 1)) / log(vocab + 1), the ranks spread over the table."""
    u = torch.rand(n, generator=g, device=DEVICE, dtype=torch.float64)
    rank = ((vocab + 1.0) ** u).floor().to(torch.int64).sub_(1).clamp_(0, vocab - 1)
    return torch.randperm(vocab, generator=g, device=DEVICE)[rank]


def _expected_rows(n, vocab):
    """Distinct rows that n such tokens are expected to name."""
    k = torch.arange(vocab, dtype=torch.float64)
    p = torch.log((k + 2) / (k + 1)) / math.log(vocab + 1)
    return float((1.0 - torch.exp(n * torch.log1p(-p))).sum())


def _tensor_sizes(case):
    if case["layout"] == "mlp":
        return [784 * 512, 512, 512 * 128, 128, 128 * 10, 10]
    if case["layout"] == "decoder":
        layer = [Q_DIM * HIDDEN, KV_DIM * HIDDEN, KV_DIM * HIDDEN, Q_DIM * HIDDEN, INTER * HIDDEN, INTER * HIDDEN,
                 INTER * HIDDEN, HIDDEN, HIDDEN, HEAD_DIM, HEAD_DIM]
        return [VOCAB * HIDDEN, *(layer * LAYERS), HIDDEN, VOCAB * HIDDEN]
    # a few large matrices, many small ones, vectors of a few elements
    g = torch.Generator().manual_seed(case["tensors"] * 7919 + case["elements"])
    share = torch.exp(3.0 * torch.randn(case["tensors"], generator=g, dtype=torch.float64))
    sizes = (share / share.sum() * case["elements"]).floor().to(torch.int64).clamp_(1)
    return [int(v) for v in sizes]


def _sequences(case, g):
    """Row offsets of ragged sequences that fill the n rows (some may be empty), and each row's sequence and place."""
    n, s = case["n"], case["seqs"]
    cuts = torch.rand(s - 1, generator=g, device=DEVICE).mul_(0.8).add_(torch.arange(1, s, device=DEVICE) - 0.4)
    cuts = cuts.mul_(n / s).round_().clamp_(0, n).to(torch.int64).sort().values
    cu = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), n)])
    row = torch.arange(n, device=DEVICE)
    seq = torch.searchsorted(cu[1:], row, right=True)
    return cu, seq, row - cu[seq], (cu[1:] - cu[:-1])[seq]


def _row_logps(logits, targets, temperature):
    out = []
    for i in range(0, logits.shape[0], 256):
        x = logits[i:i + 256].double() / temperature
        t = targets[i:i + 256].clamp_min(0)
        out.append(x.gather(1, t[:, None])[:, 0] - torch.logsumexp(x, 1))
    return torch.cat(out)


def prepare(case, seed):
    g = _generator(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] in ("lookup", "embed_grad"):
        n, vocab, hidden = case["n"], case["vocab"], case["hidden"]
        ids = _token_ids(n, vocab, g)
        if case["op"] == "lookup":
            return dict(case=case, ids=ids, table=torch.randn(vocab, hidden, generator=g, device=DEVICE, dtype=dt) * 0.02)
        st = dict(case=case, ids=ids, grad=torch.randn(n, hidden, generator=g, device=DEVICE, dtype=dt) * 0.01, out=None)
        if case["accumulate"]:
            st["out"] = torch.randn(vocab, hidden, generator=g, device=DEVICE) * 0.01
        return st
    if case["op"] in ("logps", "policy", "preference"):
        n, vocab, temp = case["n"], case["vocab"], case["temperature"]
        cu, seq, place, length = _sequences(case, g)
        targets = torch.randint(0, vocab, (n,), generator=g, device=DEVICE)
        # logits of a trained model: a wide spread, the taken token near the front
        logits = torch.randn(n, vocab, generator=g, device=DEVICE, dtype=dt) * 2.5
        front = 3.1 + math.log(vocab) - 1.0 + 1.5 * torch.randn(n, 1, generator=g, device=DEVICE)
        logits.scatter_(1, targets[:, None], front.to(dt))
        lp = None if case["op"] == "logps" else _row_logps(logits, targets, temp)
        if n > 1:
            targets = torch.where(place * 4 < length, IGNORE, targets)      # the first quarter is the prompt
        if case["op"] == "logps":
            return dict(case=case, logits=logits, targets=targets)
        ref = (lp + 0.2 * torch.randn(n, generator=g, device=DEVICE)).float()
        st = dict(case=case, logits=logits, targets=targets, ref=ref, cu=cu)
        if case["op"] == "policy":
            shift = 0.15 * torch.randn(n, generator=g, device=DEVICE, dtype=torch.float64)
            # the loss's slope jumps where exp(shift) meets a clip bound: no token sits within 1e-3 of one, where
            # the last bit of a logarithm would decide
            for edge in (math.log(0.8), math.log(1.28)):
                shift = torch.where((shift - edge).abs() < 1e-3, shift + 2e-3, shift)
            st["old"] = (lp - shift).float()
            st["adv"] = torch.randn(case["seqs"], generator=g, device=DEVICE)
        return st
    sizes = _tensor_sizes(case)
    total = sum(sizes)
    pitch = [-(-s // 64) * 64 for s in sizes]
    flat = torch.randn(sum(pitch), generator=g, device=DEVICE, dtype=dt)
    spread = torch.exp(0.5 * torch.randn(len(sizes), generator=torch.Generator().manual_seed(seed), dtype=torch.float64))
    out = torch.zeros_like(flat)
    grads, outs, at = [], [], 0
    for s, p, w in zip(sizes, pitch, spread.tolist()):
        grads.append(flat[at:at + s].mul_(8.0 * w / total ** 0.5))          # a global norm near 10
        outs.append(out[at:at + s])
        at += p
    # clipped into a second buffer, so that every pass clips the same gradients
    return dict(case=case, grads=grads, outs=outs, out=out, max_norm=1.0)


def _plain_rows(st):
    """(lp with 0 at ignored rows, valid, softmax, target column) of the logit rows."""
    valid = st["targets"] >= 0
    t = st["targets"].clamp_min(0)[:, None]
    x = st["logits"].float() / st["case"]["temperature"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    s = e.sum(1, keepdim=True)
    lp = (x.gather(1, t) - m - torch.log(s))[:, 0]
    return torch.where(valid, lp, 0.0), valid, e, s, t


def _plain_logit_grad(st, e, s, t, coef):
    """coef_r (1{j = t_r} - e[r, j] / s_r) / T, rounded once."""
    coef = (coef / st["case"]["temperature"])[:, None]
    g = e.div_(s).mul_(-coef)
    return g.scatter_add_(1, t, coef).to(st["logits"].dtype)


def _plain_policy(st):
    c = st["case"]
    lp, valid, e, s, t = _plain_rows(st)
    row = torch.arange(c["n"], device=lp.device)
    seq = torch.searchsorted(st["cu"][1:], row, right=True)
    v = valid.float()
    if c["reduction"] == "token":
        w = v / v.sum().clamp_min(1.0)
    else:
        count = torch.zeros(c["seqs"], device=lp.device).index_add_(0, seq, v)
        w = v / count.clamp_min(1.0)[seq] / (count > 0).sum().clamp_min(1)
    adv = st["adv"][seq]
    ratio = torch.exp(lp - st["old"])
    free, held = ratio * adv, ratio.clamp(1 - 0.2, 1 + 0.28) * adv
    clipped = held < free
    d = st["ref"] - lp
    kl = torch.exp(d) - d - 1.0
    loss = (w * (torch.where(valid, -torch.minimum(free, held) + c["kl_coef"] * kl, 0.0))).sum()
    coef = torch.where(valid, w * (torch.where(clipped, 0.0, -free) + c["kl_coef"] * (1.0 - torch.exp(d))), 0.0)
    return {"loss": loss, "logps": lp, "kl": (w * torch.where(valid, kl, 0.0)).sum(),
            "clip_fraction": (w * clipped).sum(), "grad": _plain_logit_grad(st, e, s, t, coef)}


def _plain_preference(st):
    c = st["case"]
    lp, valid, e, s, t = _plain_rows(st)
    row = torch.arange(c["n"], device=lp.device)
    seq = torch.searchsorted(st["cu"][1:], row, right=True)
    pairs = c["seqs"] // 2
    d = torch.zeros(c["seqs"], device=lp.device).index_add_(0, seq, torch.where(valid, lp - st["ref"], 0.0))
    chosen, rejected = 0.1 * d[:pairs], 0.1 * d[pairs:]
    h = chosen - rejected
    eps = c["smoothing"]
    soft = torch.log1p(torch.exp(-h.abs()))
    loss = ((1 - eps) * (soft + (-h).clamp_min(0.0)) + eps * (soft + h.clamp_min(0.0))).mean()
    slope = -(1 - eps) / (1.0 + torch.exp(h)) + eps / (1.0 + torch.exp(-h))
    side = torch.cat([slope, -slope]) * (0.1 / pairs)
    coef = torch.where(valid, side[seq], 0.0)
    return {"loss": loss, "chosen_rewards": chosen, "rejected_rewards": rejected, "logps": lp,
            "grad": _plain_logit_grad(st, e, s, t, coef)}


def _plain(st):
    c = st["case"]
    if c["op"] == "lookup":
        return (st["table"][st["ids"]].float() * c["scale"]).to(st["table"].dtype)
    if c["op"] == "embed_grad":
        g = st["grad"].float() * c["scale"]
        if c["accumulate"]:
            return st["out"].index_add_(0, st["ids"], g)
        return torch.zeros(c["vocab"], c["hidden"], device=g.device).index_add_(0, st["ids"], g).to(st["grad"].dtype)
    if c["op"] == "logps":
        return _plain_rows(st)[0]
    if c["op"] == "policy":
        return _plain_policy(st)
    if c["op"] == "preference":
        return _plain_preference(st)
    norm = torch.stack([g.float().square().sum() for g in st["grads"]]).sum().sqrt()
    coef = (st["max_norm"] / (norm + 1e-6)).clamp_max(1.0)
    [o.copy_(g.float() * coef) for o, g in zip(st["outs"], st["grads"])]
    return {"norm": norm, "clipped": st["out"]}


def run(state):
    if not own:
        return _plain(state)
    from memintelli_flash_b200 import NN_layers, tuning
    c, st = state["case"], state
    if c["op"] == "lookup":
        return NN_layers.embedding_scaled(st["ids"], st["table"], c["scale"])
    if c["op"] == "embed_grad":
        return NN_layers.embedding_scaled_grad(st["ids"], st["grad"], c["vocab"], c["scale"], out=st["out"],
                                               accumulate=c["accumulate"])
    if c["op"] == "logps":
        return tuning.token_logprobs(st["logits"], st["targets"], temperature=c["temperature"])
    if c["op"] == "policy":
        r, grad = tuning.policy_loss_grad(st["logits"], st["targets"], st["old"], st["adv"], st["ref"],
                                          cu_seqlens=st["cu"], clip_low=0.2, clip_high=0.28, kl_coef=c["kl_coef"],
                                          reduction=c["reduction"], temperature=c["temperature"])
        return {"loss": r.loss, "logps": r.logps, "kl": r.kl, "clip_fraction": r.clip_fraction, "grad": grad}
    if c["op"] == "preference":
        r, grad = tuning.preference_loss_grad(st["logits"], st["targets"], st["ref"], cu_seqlens=st["cu"], beta=0.1,
                                              label_smoothing=c["smoothing"], temperature=c["temperature"])
        return {"loss": r.loss, "chosen_rewards": r.chosen_rewards, "rejected_rewards": r.rejected_rewards,
                "logps": r.logps, "grad": grad}
    norm = tuning.clip_grad_norm_(st["grads"], st["max_norm"], out=st["outs"])
    return {"norm": norm, "clipped": st["out"]}


def work(case):
    """Bytes of the inputs read once and the outputs written once; the operations of the formulas."""
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "lookup":
        n, h = case["n"], case["hidden"]
        return {"bytes": size * h * (n + _expected_rows(n, case["vocab"])) + 8 * n, "flops": n * h}
    if case["op"] == "embed_grad":
        n, h = case["n"], case["hidden"]
        rows = 8 * h * _expected_rows(n, case["vocab"]) if case["accumulate"] else size * h * case["vocab"]
        return {"bytes": size * n * h + rows + 8 * n, "flops": 2 * n * h}
    if case["op"] in ("logps", "policy", "preference"):
        n, v = case["n"], case["vocab"]
        read = 0.75 * n if n > 1 else n                 # a prompt row's logits are not needed, its gradient is zero
        written = 0 if case["op"] == "logps" else n
        return {"bytes": size * v * (read + written) + 24 * n, "flops": 5 * read * v + 3 * written * v}
    return {"bytes": 2 * size * case["elements"], "flops": 3 * case["elements"]}


def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "lookup":
        return torch.index_select(st["table"], 0, st["ids"]).to(f64) * case["scale"]
    if case["op"] == "embed_grad":
        order = torch.argsort(st["ids"], stable=True)
        ids, rows = st["ids"][order], st["grad"].to(f64)[order]
        total = torch.cumsum(rows, 0)
        last = torch.ones_like(ids, dtype=torch.bool)
        last[:-1] = ids[1:] != ids[:-1]
        sums = total[last]
        sums[1:] -= total[last][:-1]
        dw = torch.zeros(case["vocab"], case["hidden"], dtype=f64, device=DEVICE) if st["out"] is None else st["out"].to(f64)
        dw[ids[last]] += case["scale"] * sums
        return dw
    if case["op"] == "clip":
        ss = sum(torch.dot(g.to(f64), g.to(f64)).item() for g in st["grads"])
        norm = math.sqrt(ss)
        k = min(1.0, st["max_norm"] / (norm + 1e-6))
        flat = torch.zeros(st["out"].numel(), dtype=f64, device=DEVICE)
        at = 0
        for g in st["grads"]:
            flat[at:at + g.numel()] = g.to(f64) * k
            at += -(-g.numel() // 64) * 64
        return {"norm": torch.tensor(norm, dtype=f64), "clipped": flat}
    # the two losses: row quantities first, then sums over sequences on the host
    n, temp = case["n"], case["temperature"]
    targets = st["targets"]
    keep = targets != IGNORE
    lp = torch.where(keep, _row_logps(st["logits"], targets, temp), 0.0)
    if case["op"] == "logps":
        return lp
    slope, cu = torch.zeros(n, dtype=f64, device=DEVICE), st["cu"].tolist()
    spans = [(a, b, int(keep[a:b].sum())) for a, b in zip(cu[:-1], cu[1:])]
    ref = st["ref"].to(f64)
    out = {"logps": lp}
    if case["op"] == "policy":
        total, live = sum(k for _, _, k in spans), sum(k > 0 for _, _, k in spans)
        loss = kl = cf = 0.0
        for (a, b, k), adv in zip(spans, st["adv"].tolist()):
            if k == 0:
                continue
            w = keep[a:b].to(f64) / (total if case["reduction"] == "token" else k * live)
            r = torch.exp(lp[a:b] - st["old"][a:b].to(f64))
            bound = 1.28 if adv > 0 else 0.8
            over = r > bound if adv > 0 else r < bound
            gain = adv * torch.where(over, bound, r)
            u = torch.exp(ref[a:b] - lp[a:b])
            k3 = u - 1 - (ref[a:b] - lp[a:b])
            loss += float((w * (case["kl_coef"] * k3 - gain)).sum())
            kl += float((w * k3).sum())
            cf += float((w * over).sum())
            slope[a:b] = w * (case["kl_coef"] * (1 - u) - torch.where(over, 0.0, adv * r))
        out.update(loss=torch.tensor(loss, dtype=f64), kl=torch.tensor(kl, dtype=f64), clip_fraction=torch.tensor(cf, dtype=f64))
    else:
        pairs, eps = case["seqs"] // 2, case["smoothing"]
        delta = [0.1 * float(((lp[a:b] - ref[a:b]) * keep[a:b]).sum()) for a, b, _ in spans]
        loss = 0.0
        for i in range(pairs):
            h = delta[i] - delta[pairs + i]
            sig = 0.5 * (1.0 + math.tanh(0.5 * h))
            loss += ((1 - eps) * math.log1p(math.exp(-h)) + eps * math.log1p(math.exp(h))) / pairs
            k = 0.1 / pairs * (sig - (1 - eps))
            for s, c in ((i, k), (pairs + i, -k)):
                a, b, _ = spans[s]
                slope[a:b] = c * keep[a:b]
        out.update(loss=torch.tensor(loss, dtype=f64), chosen_rewards=torch.tensor(delta[:pairs], dtype=f64),
                   rejected_rewards=torch.tensor(delta[pairs:], dtype=f64))
    grad = torch.empty(n, case["vocab"], dtype=f64, device=DEVICE)
    for i in range(0, n, 256):
        c = (slope[i:i + 256] / temp)[:, None]
        g = torch.softmax(st["logits"][i:i + 256].to(f64) / temp, 1) * -c
        grad[i:i + 256] = g.scatter_add_(1, targets[i:i + 256].clamp_min(0)[:, None], c)
    out["grad"] = grad
    return out
