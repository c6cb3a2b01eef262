"""What the loss and update operators are measured on: the cases, their plain forms in elementary torch operations, and
their values in 64 bits.

    token_logprobs   log-probabilities of given tokens under rows of logits, and the gradient of the logits
    preference       paired log ratios of preferred and rejected responses: loss, rewards and gradient
    policy           clipped importance ratios with a KL term: loss, statistics and gradient
    orthogonalize    a matrix update brought near its polar factor by an odd polynomial of products
"""
import math

import torch

own = False  # True: run() calls the framework's kernels

DTYPES = {"float64": torch.float64, "float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
NS = (3.4445, -4.7750, 2.0315)  # the default polynomial a s + b s^3 + c s^5
IGNORE = -100


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # scoring the rows of one decoding step of a small batch: nothing but latency
        dict(name="logprobs step", op="logprobs", rows=8, vocab=32000, pad=0, shift=0, ignored=0.0, temperature=1.0, grad=False, dtype="bfloat16"),
        # a training batch of a few documents whose logits are shifted against their tokens (a view with two strides), odd vocabulary
        dict(name="logprobs shifted odd", op="logprobs", rows=1020, vocab=50001, pad=0, shift=4, ignored=0.25, temperature=1.0, grad=True, dtype="float32"),
        # a training step's packed tokens
        dict(name="logprobs train", op="logprobs", rows=8192, vocab=32768, pad=0, shift=0, ignored=0.1, temperature=1.0, grad=True, dtype="bfloat16"),
        # scoring a rollout batch under a fixed model with a large vocabulary, at the sampling temperature
        dict(name="logprobs score wide", op="logprobs", rows=8192, vocab=131072, pad=64, shift=0, ignored=0.0, temperature=0.7, grad=False, dtype="bfloat16"),
        # a micro batch of short answers
        dict(name="preference small", op="preference", pairs=4, longest=60, packed=True, masked=0.0, kind="logistic", smoothing=0.0, normalize=False, dtype="float32"),
        # a padded batch with prompts masked out and smoothed labels
        dict(name="preference padded", op="preference", pairs=256, longest=2047, packed=False, masked=0.3, kind="logistic", smoothing=0.1, normalize=False, dtype="float32"),
        # few, very long answers: one sequence has to be shared by many workgroups; lengths normalised
        dict(name="preference long", op="preference", pairs=24, longest=131072, packed=True, masked=0.1, kind="squared", smoothing=0.0, normalize=True, dtype="float32"),
        # one group of short rollouts, an advantage for each of them
        dict(name="policy small", op="policy", seqs=16, longest=200, packed=True, masked=0.0, per_token=False, kl=0.0, reduction="sequences", dtype="float32"),
        # a large rollout batch with a reference, an advantage for each token and tool outputs masked out
        dict(name="policy large", op="policy", seqs=2048, longest=8192, packed=True, masked=0.2, per_token=True, kl=0.05, reduction="tokens", dtype="float32"),
        # the update of one small projection
        dict(name="orthogonalize small", op="orthogonalize", batch=1, rows=128, cols=256, steps=5, dtype="float32"),
        # a stack of expanding projections, kept and updated in 16 bits
        dict(name="orthogonalize stack", op="orthogonalize", batch=4, rows=1024, cols=4096, steps=5, dtype="bfloat16"),
        # one large square projection in 32 bits, its sides not multiples of any tile
        dict(name="orthogonalize large", op="orthogonalize", batch=1, rows=4000, cols=4100, steps=5, dtype="float32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("logprobs", "preference", "policy", "orthogonalize"))
    if op == "logprobs":
        vocab = _log(rng, 500, 160000)
        shift = rng.choice((0, 0, 3))
        rows = _log(rng, 1, min(16384, (1 << 29) // vocab))
        rows = max(rows // shift, 1) * shift if shift else rows
        return dict(op=op, rows=rows, vocab=vocab, pad=rng.choice((0, 0, 1, 24)), shift=shift,
                    ignored=rng.choice((0.0, 0.2)), temperature=rng.choice((1.0, 1.0, 0.6, 1.3)), grad=rng.random() < 0.6,
                    dtype=rng.choice(("bfloat16", "bfloat16", "float32", "float16", "float64")))
    if op == "preference":
        longest = _log(rng, 2, 65536)
        return dict(op=op, pairs=_log(rng, 1, min(2048, (1 << 23) // longest)), longest=longest, packed=rng.random() < 0.5,
                    masked=rng.choice((0.0, 0.1, 0.5)), kind=rng.choice(("logistic", "logistic", "hinge", "squared")),
                    smoothing=rng.choice((0.0, 0.1)), normalize=rng.random() < 0.4, dtype=rng.choice(("float32", "float32", "float64", "bfloat16")))
    if op == "policy":
        longest = _log(rng, 2, 32768)
        return dict(op=op, seqs=_log(rng, 1, min(4096, (1 << 23) // longest)), longest=longest, packed=rng.random() < 0.5,
                    masked=rng.choice((0.0, 0.1, 0.5)), per_token=rng.random() < 0.5, kl=rng.choice((0.0, 0.01, 0.1)),
                    reduction=rng.choice(("tokens", "sequences")), dtype=rng.choice(("float32", "float32", "float64", "bfloat16")))
    rows, cols = _log(rng, 16, 2000), _log(rng, 16, 5000)
    batch = rng.choice((1, 1, _log(rng, 2, 16)))
    while batch > 1 and batch * min(rows, cols) ** 2 * max(rows, cols) > 2 ** 34:
        batch //= 2
    return dict(op=op, batch=batch, rows=rows, cols=cols, steps=rng.choice((5, 5, 3, 6)), dtype=rng.choice(("bfloat16", "float32", "float16")))


# ------------------------------------------------------------------------------------ inputs
def _device():
    return "cuda" if torch.cuda.is_available() else "cpu"


def _lengths(case, count, rng):
    """Response lengths: spread evenly between one token and the longest, in an order of the seed's; among many an empty
    response now and then."""
    lengths = torch.linspace(1, case["longest"], count, device=rng.device).long()
    if count >= 16:
        lengths[::16] = 0
    return lengths[torch.randperm(count, generator=rng, device=rng.device)]


def _tokens(case, count, rng):
    """-> (shape of the token tensors, offsets or None, mask or None): packed responses or a padded batch."""
    dev, longest = rng.device, case["longest"]
    lengths = _lengths(case, count, rng)
    if case["packed"]:
        offsets = torch.zeros(count + 1, dtype=torch.int64, device=dev)
        offsets[1:] = lengths.cumsum(0)
        shape = (int(offsets[-1]),)
        mask = torch.rand(shape, generator=rng, device=dev) >= case["masked"] if case["masked"] else None
        return shape, offsets, mask
    shape = (count, longest)
    mask = torch.arange(longest, device=dev)[None, :] < lengths[:, None]
    if case["masked"]:
        mask &= torch.rand(shape, generator=rng, device=dev) >= case["masked"]
    return shape, None, mask


def _logps(shape, rng):
    """Log-probabilities as a trained model gives them: most near zero, some far below."""
    u = torch.rand(shape, generator=rng, device=rng.device)
    return -(-torch.log(u.clamp_min(1e-6))).pow(2) * 0.5


def prepare(case, seed):
    dev = _device()
    rng = torch.Generator(device=dev)
    rng.manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=rng, device=dev)  # noqa: E731
    dt = DTYPES[case["dtype"]]
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        full = rows if not case["shift"] else rows + case["shift"]  # a row more for each of `shift` documents
        logits = torch.empty(full, vocab + case["pad"], dtype=dt, device=dev)
        for at in range(0, full, 4096):  # (in pieces: the 32-bit values of a wide batch would not be small)
            part = logits[at:at + 4096]
            part.copy_(randn(*part.shape) * 2.0)
        targets = torch.randint(0, vocab, (full,), generator=rng, device=dev)
        logits[torch.arange(full, device=dev), targets] += 6.0  # the model has learnt something
        if case["ignored"]:
            targets[torch.rand(full, generator=rng, device=dev) < case["ignored"]] = IGNORE
        logits = logits[:, :vocab]
        g = randn(rows).float() / rows
        if case["shift"]:
            docs = case["shift"]
            logits = logits.reshape(docs, full // docs, vocab)[:, :-1]
            targets = targets.reshape(docs, full // docs)[:, 1:].contiguous()
            g = g.reshape(targets.shape)
        return {"case": case, "logits": logits, "targets": targets, "grad": g.to(torch.float64) if dt == torch.float64 else g}
    if case["op"] == "preference":
        shape, offsets, mask = _tokens(case, 2 * case["pairs"], rng)
        ref = _logps(shape, rng)
        logps = (ref + 0.2 * randn(*shape)).clamp_max(0.0)
        return {"case": case, "logps": logps.to(dt), "ref": ref.to(dt), "offsets": offsets, "mask": mask}
    if case["op"] == "policy":
        shape, offsets, mask = _tokens(case, case["seqs"], rng)
        old = _logps(shape, rng)
        logps = (old + 0.15 * randn(*shape)).clamp_max(0.0)
        ref = (old + 0.2 * randn(*shape)).clamp_max(0.0).to(dt) if case["kl"] else None
        adv = randn(*(shape if case["per_token"] else (case["seqs"],)))
        return {"case": case, "logps": logps.to(dt), "old": old.to(dt), "ref": ref, "advantages": adv.to(dt), "offsets": offsets, "mask": mask}
    b, m, n = case["batch"], case["rows"], case["cols"]
    r = max(1, min(m, n) // 8)  # a gradient: a part of low rank, and what a batch's samples add to it
    g = randn(b, m, r) @ randn(b, r, n) / math.sqrt(r) + 0.3 * randn(b, m, n)
    g = (g * 1e-3).to(dt)
    return {"case": case, "update": g if b > 1 else g[0]}


# ------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        from rust_lbfgs_amd import directions, losses

        if case["op"] == "logprobs":
            kw = dict(temperature=case["temperature"], ignore_index=IGNORE)
            if not case["grad"]:
                return losses.token_logprobs(state["logits"], state["targets"], **kw)
            logps, lse = losses.token_logprobs_with_lse(state["logits"], state["targets"], **kw)
            return logps, losses.token_logprobs_grad(state["logits"], state["targets"], lse, state["grad"], **kw)
        if case["op"] == "preference":
            smoothing = case["smoothing"] if case["kind"] == "logistic" else 0.0  # the other kinds have none
            r = losses.preference(state["logps"], state["ref"], offsets=state["offsets"], mask=state["mask"], beta=0.1, kind=case["kind"],
                                  label_smoothing=smoothing, normalize_lengths=case["normalize"])
            return r.f, r.rewards, r.grad
        if case["op"] == "policy":
            advantages = state["advantages"] if case["per_token"] else state["advantages"].unsqueeze(1)  # [sequences, 1]: one for each
            r = losses.policy(state["logps"], state["old"], advantages, ref_logps=state["ref"], offsets=state["offsets"],
                              mask=state["mask"], clip_low=0.2, clip_high=0.28, kl_coef=case["kl"], reduction=case["reduction"])
            return r.f, r.kl, r.clip_fraction, r.grad
        return directions.orthogonalize(state["update"], steps=case["steps"], coefficients=NS)
    plain = {"logprobs": _plain_logprobs, "preference": _plain_preference, "policy": _plain_policy, "orthogonalize": _plain_orthogonalize}
    return plain[case["op"]](state)


def _wide(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def _plain_logprobs(state):
    case, logits, targets = state["case"], state["logits"], state["targets"]
    x = logits.to(_wide(logits.dtype)) / case["temperature"]
    live = targets != IGNORE
    at = torch.where(live, targets, 0).unsqueeze(-1)
    e = x - x.amax(-1, keepdim=True)
    chosen = e.gather(-1, at)
    e = e.exp()
    total = e.sum(-1, keepdim=True)
    logps = torch.where(live, (chosen - total.log()).squeeze(-1), 0.0)
    if not case["grad"]:
        return logps
    g = torch.where(live, state["grad"], 0.0).unsqueeze(-1) / case["temperature"]
    dlogits = e * (-g / total)
    dlogits.scatter_add_(-1, at, g)
    return logps, dlogits.to(logits.dtype)


def _rows(values, offsets, mask):
    """Padded batches and packed responses alike: -> (flat values' sequence numbers, kept places, places of the sequences)."""
    if offsets is None:
        count, longest = values.shape
        offsets = torch.arange(count + 1, device=values.device) * longest
    count = offsets.numel() - 1
    seq = torch.repeat_interleave(torch.arange(count, device=values.device), offsets[1:] - offsets[:-1], output_size=values.numel())
    keep = torch.ones(values.numel(), dtype=torch.bool, device=values.device) if mask is None else mask.reshape(-1)
    return seq, keep, offsets


def _sums(values, offsets):
    """Sums over sequences, in 64 bits: thousands of terms, and differences of the sums are what matters."""
    running = torch.cat((torch.zeros(1, dtype=torch.float64, device=values.device), values.double().cumsum(0)))
    return running[offsets[1:]] - running[offsets[:-1]]


def _plain_preference(state):
    case, logps = state["case"], state["logps"]
    out = _wide(logps.dtype)
    seq, keep, offsets = _rows(logps, state["offsets"], state["mask"])
    ratio = torch.where(keep, logps.reshape(-1).double() - state["ref"].reshape(-1).double(), 0.0)
    delta = _sums(ratio, offsets)
    scale = torch.ones_like(delta)
    if case["normalize"]:
        scale = 1.0 / _sums(keep, offsets).clamp_min(1.0)
        delta = delta * scale
    pairs, beta, eps = delta.numel() // 2, 0.1, case["smoothing"]
    margin = delta[:pairs] - delta[pairs:]
    h = beta * margin
    if case["kind"] == "logistic":
        soft = torch.log1p(torch.exp(-h.abs()))
        loss = (1 - eps) * (soft + (-h).clamp_min(0.0)) + eps * (soft + h.clamp_min(0.0))
        slope = beta * (eps - 1.0 / (1.0 + torch.exp(h)))
    elif case["kind"] == "hinge":
        loss = (1.0 - h).clamp_min(0.0)
        slope = -beta * (h < 1.0).double()
    else:
        loss = (margin - 0.5 / beta).square()
        slope = 2.0 * (margin - 0.5 / beta)
    slope = torch.cat((slope, -slope)) * scale / pairs
    grad = torch.where(keep, slope[seq], 0.0).reshape(logps.shape)
    return (loss.sum() / pairs).to(out), (beta * delta).to(out), grad.to(logps.dtype)


def _plain_policy(state):
    case, logps = state["case"], state["logps"]
    out = _wide(logps.dtype)
    seq, keep, offsets = _rows(logps, state["offsets"], state["mask"])
    lp = logps.reshape(-1).double()  # 64 bits: ratios beside the clipping border, and a KL term that cancels
    d = lp - state["old"].reshape(-1).double()
    a = (state["advantages"].reshape(-1) if case["per_token"] else state["advantages"][seq]).double()
    ratio = d.exp()
    clipped = torch.where(a >= 0, ratio > 1.28, ratio < 0.8) & (a != 0)
    loss = -torch.minimum(ratio * a, ratio.clamp(0.8, 1.28) * a)
    slope = torch.where(clipped, 0.0, -ratio * a)
    kl = torch.zeros_like(lp)
    if case["kl"]:
        q = state["ref"].reshape(-1).double() - lp
        kl = q.expm1() - q
        loss = loss + case["kl"] * kl
        slope = slope - case["kl"] * q.expm1()
    tokens = _sums(keep, offsets)
    if case["reduction"] == "tokens":
        weight = (1.0 / tokens.sum().clamp_min(1.0)).expand_as(tokens)
    else:
        weight = 1.0 / (tokens.clamp_min(1.0) * (tokens > 0).sum().clamp_min(1))
    w = torch.where(keep, weight[seq], 0.0)
    total = tokens.sum().clamp_min(1.0)
    grad = torch.where(keep, slope * w, 0.0).reshape(logps.shape)
    return (torch.where(keep, loss * w, 0.0).sum().to(out), (torch.where(keep, kl, 0.0).sum() / total).to(out),
            ((clipped & keep).sum() / total).to(out), grad.to(logps.dtype))


def _plain_orthogonalize(state):
    g = state["update"]
    a, b, c = NS
    norm = g.double().square().sum((-2, -1), keepdim=True).sqrt()
    x = torch.where(norm > 0, g.double() / norm, 0.0).float()
    if g.shape[-2] > g.shape[-1]:
        x = x.mT.contiguous()
    steps = state["case"]["steps"]
    while steps:
        s = x @ x.mT.contiguous()
        x = a * x + (b * s + c * (s @ s)) @ x
        steps -= 1
    return (x.mT if g.shape[-2] > g.shape[-1] else x).contiguous().to(g.dtype)


# ------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = {"float64": 8, "float32": 4, "bfloat16": 2, "float16": 2}[case["dtype"]]
    wide = 8 if case["dtype"] == "float64" else 4
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        live = 1.0 - case["ignored"]  # rows without a target are not read
        moved = rows * vocab * size * live + rows * (8 + wide)
        if case["grad"]:
            moved += rows * vocab * size + rows * wide
        return {"bytes": moved, "flops": rows * vocab * live * (7.0 if case["grad"] else 4.0)}
    if case["op"] in ("preference", "policy"):
        seqs = 2 * case["pairs"] if case["op"] == "preference" else case["seqs"]
        tokens = seqs * case["longest"] * (0.5 if case["packed"] else 1.0)
        each = 3 * size if case["op"] == "preference" else (3 + (1 if case["kl"] else 0) + (1 if case["per_token"] else 0)) * size
        each += 1 if case["masked"] or not case["packed"] else 0
        return {"bytes": tokens * each + seqs * (8 + wide), "flops": tokens * (4.0 if case["op"] == "preference" else 30.0)}
    b, m, n, k = case["batch"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"]), case["steps"]
    # symmetric products have half the entries; either every step works on the matrix, or the steps work on its Gram matrix
    steps = min(k * (3.0 * m * m * n + m ** 3), 3.0 * m * m * n + (4 * k - 3) * float(m) ** 3)
    return {"bytes": 2.0 * b * m * n * size, "flops": b * steps}


# ------------------------------------------------------------------------------------ the values in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(case, state)
    if case["op"] == "orthogonalize":
        return _exact_orthogonalize(case, state)
    return (_exact_preference if case["op"] == "preference" else _exact_policy)(case, state)


def _exact_logprobs(case, state):
    targets = state["targets"]
    grad = state["grad"].reshape(-1).double()
    flat_t = targets.reshape(-1)
    logits = state["logits"]
    width = logits.shape[-2] if logits.dim() == 3 else None
    logps = torch.zeros(flat_t.numel(), dtype=torch.float64, device=flat_t.device)
    dl = torch.zeros(flat_t.numel(), case["vocab"], dtype=torch.float64, device=flat_t.device) if case["grad"] else None
    for at in range(0, flat_t.numel(), 512):
        r = torch.arange(at, min(at + 512, flat_t.numel()), device=flat_t.device)
        x = (logits[r] if width is None else logits[r // width, r % width]).double() / case["temperature"]
        p = torch.softmax(x, -1)
        t = flat_t[r]
        live = (t != IGNORE).double()
        hot = torch.zeros_like(p)
        hot[torch.arange(len(r), device=r.device), t.clamp_min(0)] = 1.0
        logps[r] = live * ((x * hot).sum(-1) - torch.logsumexp(x, -1))
        if dl is not None:
            dl[r] = (hot - p) * (live * grad[r] / case["temperature"])[:, None]
    logps = logps.reshape(targets.shape)
    return logps if dl is None else (logps, dl.reshape(*targets.shape, case["vocab"]))


def _spans(state):
    """Where each sequence's tokens are, as host numbers."""
    if state["offsets"] is not None:
        at = state["offsets"].tolist()
        return list(zip(at[:-1], at[1:]))
    count, longest = state["logps"].shape
    return [(i * longest, (i + 1) * longest) for i in range(count)]


def _kept(state):
    flat = state["logps"].reshape(-1)
    return torch.ones_like(flat, dtype=torch.float64) if state["mask"] is None else state["mask"].reshape(-1).double()


def _exact_preference(case, state):
    keep = _kept(state)
    logps, ref = state["logps"].reshape(-1).double(), state["ref"].reshape(-1).double()
    spans = _spans(state)
    delta = torch.stack([((logps[i:j] - ref[i:j]) * keep[i:j]).sum() for i, j in spans])
    per = torch.stack([keep[i:j].sum() for i, j in spans])
    inv = torch.where(per > 0, 1.0 / per, 1.0) if case["normalize"] else torch.ones_like(per)
    delta = (delta * inv).requires_grad_()
    half, beta, eps = len(spans) // 2, 0.1, case["smoothing"]
    h = beta * (delta[:half] - delta[half:])
    if case["kind"] == "logistic":
        logsig = torch.nn.functional.logsigmoid
        loss = -(1 - eps) * logsig(h) - eps * logsig(-h)
    elif case["kind"] == "hinge":
        loss = torch.relu(1.0 - h)
    else:
        loss = (h / beta - 1.0 / (2.0 * beta)) ** 2
    f = loss.mean()
    (dd,) = torch.autograd.grad(f, delta)
    grad = torch.zeros_like(logps)
    for k, (i, j) in enumerate(spans):
        grad[i:j] = dd[k] * inv[k] * keep[i:j]
    return f.detach(), (beta * delta).detach(), grad.reshape(state["logps"].shape)


def _exact_policy(case, state):
    keep = _kept(state) > 0
    logps = state["logps"].reshape(-1).double().requires_grad_()
    old, spans = state["old"].reshape(-1).double(), _spans(state)
    adv = state["advantages"].double()
    adv = adv.reshape(-1) if case["per_token"] else torch.cat([v.expand(j - i) for v, (i, j) in zip(adv, spans)])
    ratio = torch.exp(logps - old)
    over = ((adv > 0) & (ratio > 1.28)) | ((adv < 0) & (ratio < 0.8))
    bounded = torch.where(adv > 0, torch.full_like(ratio, 1.28), torch.full_like(ratio, 0.8))
    loss = -adv * torch.where(over, bounded, ratio)
    kl = torch.zeros_like(old)
    if case["kl"]:
        q = state["ref"].reshape(-1).double() - logps
        kl = torch.expm1(q) - q
        loss = loss + case["kl"] * kl
    total = max(1, int(keep.sum()))
    if case["reduction"] == "tokens":
        f = loss[keep].sum() / total
    else:
        w, some = torch.zeros_like(old), 0
        for i, j in spans:
            n = int(keep[i:j].sum())
            some += n > 0
            w[i:j] = 1.0 / max(1, n)
        f = (loss * w)[keep].sum() / max(1, some)
    (grad,) = torch.autograd.grad(f, logps)
    return f.detach(), kl[keep].detach().sum() / total, (over & keep).double().sum() / total, grad.reshape(state["logps"].shape)


def _exact_orthogonalize(case, state):
    x = state["update"].double()
    x = x.reshape(case["batch"], case["rows"], case["cols"])
    tall = case["rows"] > case["cols"]
    x = x.transpose(1, 2).contiguous() if tall else x
    a, b, c = NS
    for i in range(case["batch"]):
        y = x[i] / torch.linalg.vector_norm(x[i])
        for _ in range(case["steps"]):
            s = torch.mm(y, y.t().contiguous())
            y = torch.mm(c * torch.mm(s, s) + b * s + a * torch.eye(len(s), dtype=s.dtype, device=s.device), y)
        x[i] = y
    return (x.transpose(1, 2).contiguous() if tall else x).reshape(state["update"].shape)
