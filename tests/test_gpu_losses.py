"""Token log-probabilities, preference and policy losses on the GPU against their definitions in 64 bits.

Tolerances count roundings.  u = 2^-24 is a rounding of the 32-bit arithmetic (2^-53 of the 64-bit one), e half a step of the
result's own type.  A probability exp((x - lse)/tau) carries |x - lse|/tau roundings of its argument (scale, difference and
product: 3) and one or two of the exponential; a sum over V terms held by 64 lanes or more at least V/64 + 16 of its own."""
import math

import pytest
import torch

from rust_lbfgs_amd import LbfgsError, TorchEvaluate, lbfgs, losses

pytestmark = pytest.mark.gpu
DT = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def unit(dtype):
    """(a rounding of the arithmetic, half a step of the type, its smallest step)"""
    small = {torch.float64: 0.0, torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[dtype]
    return (2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24), torch.finfo(dtype).eps / 2, small


def near(got, want, tol, what=""):
    """Equal where not finite, else within tol (elementwise, 64 bits)."""
    got, want = got.double().cpu(), want.double().cpu()
    tol = torch.nan_to_num(torch.as_tensor(tol, dtype=torch.float64).cpu(), nan=0.0).expand_as(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    off = (got - want).abs()[fine] - tol[fine]
    assert not off.numel() or off.max() <= 0, (what, float(off.max()))


# ------------------------------------------------------------------------------------ token log-probabilities
def logprobs_in_64_bits(x, y, g, tau, ignore=-100):
    z = x.double().cpu() / tau
    y, g = y.cpu(), g.double().cpu()
    live = y != ignore
    at = torch.where(live, y, 0)
    top = z.amax(-1)
    rest = (z - top.unsqueeze(-1)).exp().sum(-1).log()
    lse = top + rest
    lp = torch.where(live, z.gather(-1, at.unsqueeze(-1)).squeeze(-1) - top - rest, 0.0)
    p = torch.softmax(z, -1)
    hot = torch.zeros_like(p).scatter_(-1, at.unsqueeze(-1), 1.0)
    use = (live & (g != 0)).unsqueeze(-1)
    return lp, torch.where(use, (g / tau).unsqueeze(-1) * (hot - p), 0.0), lse, p, live


def check_logprobs(x, y, g, tau, ignore=-100):
    u, e, small = unit(x.dtype)
    before = x.clone()
    lp, lse = losses.token_logprobs_with_lse(x, y, tau, ignore)
    dx = losses.token_logprobs_grad(x, y, lse, g, tau, ignore)
    assert torch.equal(x.view(torch.uint8) if x.is_contiguous() else x.nan_to_num(0), before.view(torch.uint8) if x.is_contiguous() else before.nan_to_num(0))
    assert lp.dtype == g.dtype and lse.dtype == torch.float64 and lse.shape == (*y.shape, 2) and dx.dtype == x.dtype and dx.shape == x.shape and dx.is_contiguous()
    wlp, wdx, wlse, p, live = logprobs_in_64_bits(x, y, g, tau, ignore)
    V = x.shape[-1]
    z = x.double().cpu() / tau
    spread = torch.nan_to_num((z - wlse.unsqueeze(-1)).abs(), nan=0.0, posinf=0.0).clamp_max(200.0)
    sums = (V / 64 + 16 + 4 * (p * spread).sum(-1)) * u  # the sum's roundings, and its terms' weighted by their size
    # x/tau of the definition as computed here is a 64-bit number, off by up to 2^-53 of its size, which is an absolute error of
    # the exponent (it shows where tau is small: |x/tau| = 1000 at 64 bits is 1e-13)
    held = 4 * 2.0 ** -53 * torch.nan_to_num(z.abs(), nan=0.0, posinf=0.0)
    held = torch.where(held < 1e-9, held, 0.0)  # (rows of the type's extreme values are exact: all of them differ by 0 or exp gives 0)
    sums = sums + (p * held).sum(-1) + held.gather(-1, torch.where(live, y.cpu(), 0).unsqueeze(-1)).squeeze(-1)
    near(lp, wlp, sums + 2 * u * (wlp.abs() + 1), "logps")
    gt = (g.double().cpu().abs() / tau).unsqueeze(-1)
    # an exponential below the smallest normal number of the arithmetic has no relative precision (in 32 bits it is 0)
    tiny = gt * torch.finfo(torch.float64 if x.dtype == torch.float64 else torch.float32).tiny
    tol = tiny + e * wdx.abs() + gt * p * ((4 * spread + 8) * u + held) + gt * p * sums.unsqueeze(-1) + small
    tol = tol + gt * sums.unsqueeze(-1) * torch.zeros_like(p).scatter_(-1, torch.where(live, y.cpu(), 0).unsqueeze(-1), 1.0)
    near(dx, wdx, tol, "dlogits")
    return lp, lse, dx


def make(rows, V, dtype, seed=0, sharp=3.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(*rows, V, generator=gen) * sharp).to(dtype).cuda()
    y = torch.randint(0, V, rows, generator=gen).cuda()
    g = torch.randn(*rows, generator=gen).to(torch.float64 if dtype == torch.float64 else torch.float32).cuda()
    return x, y, g


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows, V", [((1,), 1), ((3,), 2), ((5,), 7), ((2, 3), 8), ((4,), 63), ((70,), 1000), ((3, 1, 5), 2049), ((2,), 50001), ((300,), 4099)])
def test_logprobs_sizes(dtype, rows, V):
    check_logprobs(*make(rows, V, DT[dtype]), 1.0)


@pytest.mark.parametrize("dtype", DT)
def test_logprobs_large_vocabulary_many_rows(dtype):
    check_logprobs(*make((257,), 40001, DT[dtype]), 0.7)


@pytest.mark.parametrize("V", [16385, 131072, 160001])
def test_logprobs_row_shared_by_workgroups(V):
    for rows in (1, 2, 33):
        check_logprobs(*make((rows,), V, torch.bfloat16, sharp=5.0), 1.3)
    check_logprobs(*make((1,), V, torch.float64), 1.0)


@pytest.mark.parametrize("dtype, V", [("bf16", 200003), ("f32", 262147), ("f64", 40001), ("f16", 196609)])
def test_logprobs_long_row_shared_by_workgroups(dtype, V):
    for rows in (1, 2, 128, 129):
        check_logprobs(*make((rows,), V, DT[dtype], sharp=5.0), 1.3)


@pytest.mark.parametrize("V", [2047, 2049, 8191, 8193, 16385, 65537])
def test_logprobs_workgroups_of_every_size(V):
    """Waves, workgroups of four and of eight for a row, with few rows and many; rows of the gradient whole and shared."""
    for rows in (1, 100, 300, 1024):
        check_logprobs(*make((rows,), V, torch.bfloat16, sharp=5.0), 0.9)


@pytest.mark.parametrize("tau", [1e-2, 0.5, 3.0, 100.0])
def test_logprobs_temperature(tau):
    for dtype in DT.values():
        check_logprobs(*make((9,), 515, dtype), tau)


@pytest.mark.parametrize("dtype, taus", [("f32", (1e-37, 1e37)), ("bf16", (1e-37, 1e37)), ("f64", (1e-300, 1e300))])
def test_logprobs_extreme_temperatures(dtype, taus):
    """All the weight on the largest logit, or the same for each that is not masked; a gradient's factor 1/temperature in the upstream one."""
    x = torch.arange(16, device="cuda").to(DT[dtype])
    x[::4] = -math.inf
    y = torch.tensor([15], device="cuda")
    for tau, want in zip(taus, (0.0, -math.log(12))):
        lp, lse = losses.token_logprobs_with_lse(x[None], y, tau)
        assert abs(float(lp) - want) <= 4e-7  # a logarithm and a sum of 12 ones in 32 bits
        d = losses.token_logprobs_grad(x[None], y, lse, torch.full_like(lp, tau), tau).double()[0]
        p = torch.zeros(16, dtype=torch.float64, device="cuda")
        p[15 if want == 0 else slice(None)] = 1 if want == 0 else 1 / 12
        p[::4] = 0
        onehot = torch.nn.functional.one_hot(y[0], 16)
        # tau/tau through 32 bits, an exponential, the rounding of the result
        assert ((d - (onehot - p)).abs() <= 1e-6 + torch.finfo(x.dtype).eps / 2).all(), tau


@pytest.mark.parametrize("tau", [1.0, 0.7, 3.0])
def test_small_probabilities_have_gradients_of_full_precision(tau):
    """Of 32-bit logits, relative to each gradient: the upstream one over tau, exp(-l) and their product 3 roundings, the hardware's
    exponential 2 (an ulp), what makes up for its argument's rounding 1, the product 1.  Down to 60 powers of e, beside logits of any size."""
    u = 2.0 ** -24
    for V, shift in ((4099, 0.0), (700, 1000.3), (50001, -7.1)):
        gen = torch.Generator().manual_seed(V)
        x = (shift - 60 * tau * torch.rand(9, V, generator=gen)).cuda()
        x[0, 5:9], x[1, 3] = -math.inf, torch.finfo(torch.float32).min
        y, g = torch.randint(20, V, (9,), generator=gen).cuda(), torch.randn(9, generator=gen).cuda()
        z = x.double()
        m = z.amax(-1, keepdim=True)
        w = ((z - m) / tau).exp()
        lse = torch.cat((m, w.sum(-1, keepdim=True).log()), 1)
        dx = losses.token_logprobs_grad(x, y, lse, g, tau)
        want = -(g.double() / tau).unsqueeze(-1) * w / w.sum(-1, keepdim=True)
        off = ((dx.double() - want).abs() - 8 * u * want.abs()).scatter(-1, y.unsqueeze(-1), 0.0)
        assert off.max() <= 0, (V, float(((dx.double() - want) / want).abs().scatter(-1, y.unsqueeze(-1), 0.0).nan_to_num(0.0).max() / u))
        assert (dx[0, 5:9] == 0).all() and dx[1, 3] == 0


def test_what_comes_into_a_loss_is_not_rounded_to_16_bits():
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.randn(4, 700, generator=torch.Generator().manual_seed(0)).cuda().to(dtype).requires_grad_()
        up = torch.tensor(1 / 3, device="cuda")
        losses.preference_loss(x).backward(up)
        want = losses.preference(x.detach()).grad.double() * up.double()
        # the product in 32 bits, rounded once more
        assert ((x.grad.double() - want).abs() <= want.abs() * (torch.finfo(dtype).eps / 2 + 2.0 ** -23) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2).all()


@pytest.mark.parametrize("dtype", DT)
def test_logprobs_ignored_and_out_of_range_targets(dtype):
    x, y, g = make((12,), 999, DT[dtype])
    y[0] = y[5] = y[11] = -100
    x[5] = math.nan  # an ignored row is not looked at
    lp, _, dx = check_logprobs(x, y, g, 1.0)
    assert (lp[[0, 5, 11]] == 0).all() and (dx[[0, 5, 11]] == 0).all()
    y[1], y[2] = 999, -1
    lp, lse = losses.token_logprobs_with_lse(x, y)
    dx = losses.token_logprobs_grad(x, y, lse, g)
    assert lp[1:3].isnan().all() and dx[1:3].isnan().all() and not lp[3:].isnan().any() and not dx[3:].isnan().any()
    y[:] = 7  # any index can be the one that is ignored
    assert (losses.token_logprobs(x, y, ignore_index=7) == 0).all()


@pytest.mark.parametrize("dtype", DT)
def test_logprobs_masked_and_special_logits(dtype):
    t = DT[dtype]
    x, y, g = make((9,), 777, t)
    x[0, 100:] = -math.inf              # the vocabulary masked by infinities
    y[0] = 50
    x[1, 100:] = torch.finfo(t).min     # ... by the type's lowest value
    y[1] = 99
    x[2] = torch.finfo(t).min           # all the same: uniform
    x[3, :] = -math.inf                 # the target alone is left
    x[3, y[3]] = 1.0
    x[4, y[4]] = -math.inf              # the target is masked: log-probability -inf, gradient finite
    x[5] = torch.finfo(t).max
    x[6, 5] = math.inf                  # NaN, as the definition's
    x[7, 5] = math.nan
    x[8] = -math.inf
    lp, lse, dx = check_logprobs(x, y, g, 1.0)
    assert lp[3] == 0 and lp[4] == -math.inf and dx[4].isfinite().all()
    assert (lp[2] - -math.log(777)).abs() < 1e-6 and lp[6:].isnan().all() and dx[6:].isnan().all()


@pytest.mark.parametrize("dtype", DT)
def test_logprobs_strides(dtype):
    t = DT[dtype]
    x, _, _ = make((4, 9), 777, t)
    y = torch.randint(0, 777, (4, 8)).cuda()
    g = torch.randn(4, 8, dtype=torch.float64 if t == torch.float64 else torch.float32).cuda()
    check_logprobs(x[:, :-1], y, g, 1.0)                                # shifted against its tokens: two strides
    check_logprobs(x[:, 1:, 3:-2], (y % 772), g, 1.0)                   # rows that start anywhere
    check_logprobs(x[:, ::2][:, :4], y[:, ::2] % 777, g[:, 1::2], 1.0)  # strided targets and gradients
    check_logprobs(x.transpose(0, 1)[:8], y.t(), g.t(), 1.0)
    check_logprobs(x[:, :-1].transpose(1, 2).contiguous().transpose(1, 2), y, g, 1.0)  # logits not adjacent: copied
    big, _, _ = make((2, 3, 4), 100, t)
    check_logprobs(big[:, :, 1:, :99], torch.randint(0, 99, (2, 3, 3)).cuda(), g[:3, :6].reshape(2, 3, 3), 1.0)
    check_logprobs(x[:1, :1].expand(4, 8, 777), y, g, 1.0)              # one row under many tokens
    check_logprobs(x[0, 0], y[0, 0], g[0, 0], 1.0)


def test_logprobs_nothing_and_zero_gradients():
    x = torch.zeros(0, 7, device="cuda")
    y = torch.zeros(0, dtype=torch.int64, device="cuda")
    lp, lse = losses.token_logprobs_with_lse(x, y)
    assert lp.shape == (0,) and losses.token_logprobs_grad(x, y, lse, lp).shape == (0, 7)
    x, y, g = make((6,), 3001, torch.bfloat16)
    x[2] = math.nan
    g[2] = 0  # no gradient comes in: the row is not read
    lp, lse = losses.token_logprobs_with_lse(x, y)
    dx = losses.token_logprobs_grad(x, y, lse, g)
    assert (dx[2] == 0).all() and lp[2].isnan() and not dx[[0, 1, 3, 4, 5]].isnan().any()


def test_logprobs_beyond_32_bits():
    """Row starts beyond 2^32 elements from the first."""
    rows, V = 33001, 131072
    x = torch.empty(rows, V, dtype=torch.bfloat16, device="cuda")
    x.fill_(-3.0)
    y = torch.full((rows,), -100, dtype=torch.int64, device="cuda")
    x[-1, -1], y[-1], y[0] = 2.0, V - 1, 5
    lp = losses.token_logprobs(x, y).cpu()
    want = 5.0 - math.log((V - 1) + math.exp(5.0))
    assert abs(float(lp[-1]) - want) < 2e-5 and abs(float(lp[0]) + math.log(V)) < 2e-5 and (lp[1:-1] == 0).all()


@pytest.mark.parametrize("dtype", DT)
def test_logprobs_autograd(dtype):
    x, y, g = make((3, 5), 321, DT[dtype])
    y[1, 2] = -100
    x.requires_grad_()
    lp = losses.token_logprobs(x, y, 0.8)
    lp.backward(g)
    p, lse = losses.token_logprobs_with_lse(x, y, 0.8)
    assert torch.equal(lp.detach(), p) and torch.equal(x.grad, losses.token_logprobs_grad(x, y, lse, g, 0.8))
    x.grad = None
    (losses.token_logprobs(x, y, 0.8).expand(2, 3, 5) * g).sum().backward()  # a broadcast gradient
    assert (x.grad.double() - 2 * losses.token_logprobs_grad(x, y, lse, g, 0.8).double()).abs().max() <= 2 * unit(x.dtype)[1] * x.grad.abs().max()
    with torch.no_grad():
        assert not losses.token_logprobs(x, y).requires_grad


def test_logprobs_gradient_against_differences():
    x, y, g = make((4,), 37, torch.float64)
    lp, lse = losses.token_logprobs_with_lse(x, y, 1.5)
    dx = losses.token_logprobs_grad(x, y, lse, g, 1.5)
    h = 2.0 ** -17
    for r, v in ((0, int(y[0])), (1, 3), (2, int(y[2])), (3, 36)):
        up, down = x.clone(), x.clone()
        up[r, v] += h
        down[r, v] -= h
        slope = ((losses.token_logprobs(up, y, 1.5) - losses.token_logprobs(down, y, 1.5)) * g).sum() / (2 * h)
        assert abs(float(slope - dx[r, v])) <= h * h * abs(float(g[r])) + 1e-15 * 200 / h  # third derivative / 6 < 1; roundings over 2 h


# ------------------------------------------------------------------------------------ sequences
def ragged(lengths, dtype, seed=0, layout="packed", masked=0.0, slack=0, bits=64):
    """-> logps, other, offsets, mask, spans in the flat tensors; masked places hold NaN."""
    gen = torch.Generator().manual_seed(seed)
    if layout == "packed":
        off = [slack]
        for n in lengths:
            off.append(off[-1] + n)
        T, spans = off[-1] + slack, list(zip(off[:-1], off[1:]))
        offsets = torch.tensor(off, dtype=torch.int64 if bits == 64 else torch.int32).cuda()
        shape = (T,)
        mask = torch.ones(T, dtype=torch.bool)
    else:
        L = max(max(lengths), 1)
        T, shape, offsets = L * len(lengths), (len(lengths), L), None
        spans = [(i * L, i * L + L) for i in range(len(lengths))]
        mask = (torch.arange(L)[None] < torch.tensor(lengths)[:, None]).reshape(-1)
    if masked:
        mask &= torch.rand(T, generator=gen) >= masked
    lp = -torch.rand(T, generator=gen) * 4
    other = (lp + 0.2 * torch.randn(T, generator=gen)).clamp_max(0)
    use_mask = masked > 0 or layout == "padded"
    keep = torch.zeros(T, dtype=torch.bool)
    for i, j in spans:
        keep[i:j] = mask[i:j]
    lp, other = lp.to(dtype), other.to(dtype)
    lp[~keep], other[~keep] = math.nan, math.inf
    return (lp.reshape(shape).cuda(), other.reshape(shape).cuda(), offsets, mask.reshape(shape).cuda() if use_mask else None, spans, keep)


def preference_in_64_bits(lp, ref, spans, keep, beta, kind, eps, normalize):
    lp, ref = lp.reshape(-1).double().cpu(), None if ref is None else ref.reshape(-1).double().cpu()
    d = torch.where(keep, lp if ref is None else lp - ref, 0.0)
    R = torch.stack([d[i:j].sum() for i, j in spans])
    n = torch.stack([keep[i:j].sum() for i, j in spans]).double()
    inv = 1.0 / n.clamp_min(1.0) if normalize else torch.ones_like(n)
    R = (R * inv).requires_grad_()
    P = len(spans) // 2
    D = R[:P] - R[P:]
    h = beta * D
    ls = torch.nn.functional.logsigmoid
    loss = {"logistic": lambda: -(1 - eps) * ls(h) - eps * ls(-h), "hinge": lambda: torch.relu(1 - h), "squared": lambda: (D - 0.5 / beta) ** 2}[kind]()
    (dR,) = torch.autograd.grad(loss.mean(), R)
    grad = torch.zeros_like(lp)
    for k, (i, j) in enumerate(spans):
        grad[i:j] = torch.where(keep[i:j], dR[k] * inv[k], 0.0)
    size = torch.stack([d[i:j].abs().sum() for i, j in spans]) * inv
    return loss.mean().detach(), beta * R.detach(), grad, size.max()


LENGTHS = {"pair": [1, 1], "empty": [0, 0], "short": [5, 0, 1, 17, 3, 2], "chunk": [2048, 2047, 1, 2049, 8, 4096], "long": [9000, 1, 0, 12345],
           "many": [(7 * k) % 13 for k in range(1200)], "ones": [1] * 4000, "wide": [(977 * k) % 5000 for k in range(40)]}


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("layout", ["packed", "padded"])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_preference(lengths, layout, dtype):
    t = DT[dtype]
    u, e, small = unit(t)
    for k, (kind, eps) in enumerate((("logistic", 0.0), ("logistic", 0.2), ("hinge", 0.0), ("squared", 0.0))):
        masked, normalize, slack, bits = (0.0, 0.4)[k % 2], k in (1, 3), (0, 3)[k // 2], (64, 32)[k % 2]
        lp, ref, off, mask, spans, keep = ragged(LENGTHS[lengths], t, 10 + k, layout, masked, slack if layout == "packed" else 0, bits)
        r = ref if k != 2 else None
        beta = (0.1, 0.5, 0.02, 1.0)[k]
        got = losses.preference(lp, r, offsets=off, mask=mask, beta=beta, kind=kind, label_smoothing=eps, normalize_lengths=normalize)
        f, rewards, grad, size = preference_in_64_bits(lp, r, spans, keep, beta, kind, eps, normalize)
        what = (lengths, layout, dtype, kind)
        wide = 2.0 ** -53 if t == torch.float64 else 2.0 ** -24
        sums = 1e-15 * (1 + float(size)) * 4  # 64-bit sums of 10^4 terms, in another order
        assert got.f.dtype == got.rewards.dtype == (torch.float64 if t == torch.float64 else torch.float32) and got.grad.dtype == t
        # the loss moves with R by at most its slope (beta, or 2 |D - 1/(2 beta)|); its own arithmetic takes a few 64-bit roundings
        slope = max(beta, 2 * (2 * float(size) + 0.5 / beta)) if kind == "squared" else beta
        near(got.f, f, wide * f.abs() + slope * sums + 1e-15 * f.abs() * 8, what)
        near(got.rewards, rewards, wide * rewards.abs() + beta * sums + 1e-15 * rewards.abs(), what)
        curve = 2.0 if kind == "squared" else beta * beta
        near(got.grad.reshape(-1), grad, (e + u) * grad.abs() * 1.01 + curve * sums + 1e-15 * grad.abs() * 8 + small, what)
        assert (got.grad.reshape(-1).cpu()[~keep] == 0).all()


@pytest.mark.parametrize("count", [64, 128, 130])
def test_preference_of_many_long_sequences(count, monkeypatch):
    """More than four chunks each: their records are added up by groups of lanes, where slopes are wanted or in a pass of its own."""
    monkeypatch.setitem(LENGTHS, "many long", [8250 + 13 * (k % 17) for k in range(count)])
    test_preference("many long", "packed", "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lengths", [[20] * 999 + [300001], [300001] + [3] * 1400 + [0], [7] * 100 + [40000, 0] + [1] * 98])
def test_one_very_long_sequence_among_many_short(lengths, dtype, monkeypatch):
    """The mean length is short, so one lane adds up the records of the long one's chunks."""
    monkeypatch.setitem(LENGTHS, "one long", lengths)
    test_preference("one long", "packed", dtype)
    test_policy("one long", "packed", dtype)


def test_preference_extreme_margins():
    """Margins far beyond where exp overflows, and an infinite one."""
    lp = torch.tensor([[0.0], [-2e4], [-1e30], [-math.inf], [-2e4], [0.0], [0.0], [0.0]], dtype=torch.float64).cuda()
    r = losses.preference(lp, beta=1.0)
    # margins 2e4, -2e4, -1e30, -inf
    assert r.f == math.inf
    assert r.grad.reshape(-1).tolist() == [0.0, -0.25, -0.25, -0.25, 0.0, 0.25, 0.25, 0.25]
    r = losses.preference(lp[[0, 1, 4, 5]], beta=1.0)
    assert float(r.f) == 1e4 and r.rewards.tolist() == [0.0, -2e4, -2e4, 0.0]
    # a NaN stays with its pair
    lp[3] = math.nan
    r = losses.preference(lp, beta=1.0)
    assert r.f.isnan() and r.grad.reshape(-1).isnan().tolist() == [False, False, False, True] * 2


def policy_in_64_bits(lp, old, adv, ref, spans, keep, low, high, kl_coef, reduction):
    x = lp.reshape(-1).double().cpu().requires_grad_()
    old = old.reshape(-1).double().cpu()
    adv = adv.double().cpu()
    if adv.shape == (len(spans), 1) and tuple(adv.shape) != tuple(lp.shape):
        full = torch.zeros_like(old)
        for k, (i, j) in enumerate(spans):
            full[i:j] = adv[k, 0]
        adv = full
    adv = adv.reshape(-1)
    xs, os_, a = x[keep], old[keep], adv[keep]
    r = torch.exp(xs - os_)
    over = ((a > 0) & (r > 1 + high)) | ((a < 0) & (r < 1 - low))
    flat = torch.where(a > 0, torch.full_like(r, 1 + high), torch.full_like(r, 1 - low))
    loss = -torch.where(over, flat, r) * a
    q = ref.reshape(-1).double().cpu()[keep] - xs if kl_coef else torch.zeros_like(xs)
    k3 = torch.expm1(q) - q
    loss = loss + kl_coef * k3
    w = torch.zeros_like(old)
    some = max(1, sum(bool(keep[i:j].any()) for i, j in spans))
    for i, j in spans:
        w[i:j] = 1.0 / (max(1, int(keep[i:j].sum())) * some)
    if reduction == "tokens":
        w = torch.full_like(old, 1.0 / max(1, int(keep.sum())))
    f = (loss * w[keep]).sum()
    (grad,) = torch.autograd.grad(f, x)
    N = max(1, int(keep.sum()))
    # what the gradient is made of, for the tolerance
    parts = torch.zeros_like(old)
    parts[keep] = ((torch.where(over, 0.0, r * a).abs() + abs(kl_coef) * (1 + q.exp())) * w[keep]).detach()
    return (f.detach(), k3.detach().sum() / N, over.double().sum() / N, grad, parts, (loss.abs() * w[keep]).detach().sum(),
            abs(kl_coef) * (k3 * w[keep]).detach().sum(), (torch.where(over, 0.0, (r - 1) * a).abs() * w[keep]).detach().sum())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("layout", ["packed", "padded"])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_policy(lengths, layout, dtype):
    t = DT[dtype]
    u, e, small = unit(t)
    for k, (reduction, kl_coef, per_token) in enumerate((("tokens", 0.0, True), ("sequences", 0.1, False), ("tokens", 0.02, False), ("sequences", 0.0, True))):
        masked, slack, bits = (0.0, 0.4)[k % 2], (0, 5)[k // 2], (64, 32)[k % 2]
        lp, old, off, mask, spans, keep = ragged(LENGTHS[lengths], t, 20 + k, layout, masked, slack if layout == "packed" else 0, bits)
        gen = torch.Generator().manual_seed(k)
        ref = (torch.nan_to_num(lp.float().cpu(), nan=0.0) + 0.7 * torch.randn(lp.shape, generator=gen)).to(t).cuda() if kl_coef else None
        adv = torch.randn(lp.shape if per_token else (len(spans), 1), generator=gen).to(t).cuda()
        adv.reshape(-1)[::7] = 0
        low, high = (0.2, 0.28) if k % 2 else (0.1, 0.1)
        got = losses.policy(lp, old, adv, ref_logps=ref, offsets=off, mask=mask, clip_low=low, clip_high=high, kl_coef=kl_coef, reduction=reduction)
        f, kl, clip, grad, parts, size, klsize, beyond = policy_in_64_bits(lp, old, adv, ref, spans, keep, low, high, kl_coef, reduction)
        what = (lengths, layout, dtype, reduction, kl_coef)
        # f: its KL part has 32-bit terms (10 roundings each), and so has r - 1 (the difference's rounding, the series' four); products
        # with the advantage and all sums are 64-bit
        near(got.f, f, u * f.abs() + 10 * u * klsize + 6 * u * beyond + 1e-14 * size, what)
        near(got.kl, kl, 11 * u * kl.abs(), what)
        near(got.clip_fraction, clip, u * clip, what)
        # grad: advantage's product, KL term, their sum, the weight and its product
        near(got.grad.reshape(-1), grad, e * grad.abs() * 1.01 + 8 * u * parts + small, what)
        assert (got.grad.reshape(-1).cpu()[~keep] == 0).all()


def test_policy_borders_and_extremes():
    """Ratios on the border are not clipped; ones beside it by the smallest step are; zero advantages give nothing."""
    h, l = math.log1p(0.2), math.log1p(-0.2)
    d = torch.tensor([math.nextafter(h, 9), math.nextafter(h, -9), math.nextafter(l, -9), math.nextafter(l, 9), 800.0, -800.0, 800.0], dtype=torch.float64)
    a = torch.tensor([1.0, 1.0, -1.0, -1.0, 1.0, -1.0, 0.0], dtype=torch.float64)
    z = torch.zeros_like(d)
    r = losses.policy(d.cuda()[None], z.cuda()[None], a.cuda()[None])
    assert (r.grad[0] == 0).tolist() == [True, False, True, False, True, True, True]
    assert float(r.clip_fraction) == pytest.approx(4 / 7, rel=1e-15) and r.f.isfinite()
    r = losses.policy(d.cuda()[None, :1], z.cuda()[None, :1], a.cuda()[None, :1], clip_high=math.inf, clip_low=1.0)  # no clipping
    assert float(r.clip_fraction) == 0 and float(r.grad) == pytest.approx(-1.2, rel=1e-14)
    x = torch.tensor([[-math.inf, -1.0]], device="cuda")
    r = losses.policy(x, x, torch.ones_like(x))  # -inf - -inf
    assert r.f.isnan() and r.grad[0].isnan().tolist() == [True, False]
    r = losses.policy(x, x, torch.ones_like(x), mask=torch.tensor([[False, True]], device="cuda"))
    assert float(r.f) == -1 and r.grad.tolist() == [[0.0, -1.0]]


def test_small_kl_terms_do_not_cancel():
    lp = -torch.rand(1, 3000, generator=torch.Generator().manual_seed(1))
    ref = lp + 1e-3 * torch.randn(1, 3000, generator=torch.Generator().manual_seed(2))
    q = ref.double() - lp.double()
    want = (torch.expm1(q) - q).mean()
    r = losses.policy(lp.cuda(), lp.cuda(), torch.zeros(1, 1, device="cuda"), ref_logps=ref.cuda(), kl_coef=1.0)
    assert abs(float(r.kl) - float(want)) <= 11 * 2.0 ** -24 * float(want)


@pytest.mark.parametrize("dtype", ["f64", "f32"])
@pytest.mark.parametrize("q", [1e-12, 1e-9, 1e-6, 1e-3, 0.03, 0.2, 0.499, 0.501, 0.9, 2.0, 5.0])
def test_kl_terms_of_every_size(q, dtype):
    """e^q - 1 - q against its series in exact fractions: relative to itself, from where it is 10^-24 to where e^q is all of it."""
    from fractions import Fraction

    t = DT[dtype]
    u, e, _ = unit(t)
    for q_ in (float(torch.tensor(v, dtype=t)) for v in (q, -q, 0.7 * q, -0.7 * q)):
        x, k, term, n = Fraction(q_), Fraction(0), Fraction(1), 1
        while n <= 60:
            term = term * x / n
            k += term if n > 1 else 0
            n += 1
        z = torch.zeros(1, 7, dtype=t, device="cuda")
        r = losses.policy(z, z, z, ref_logps=z + q_, kl_coef=1.0)
        # the exponential's rounding and the difference's beside it (|e^q - 1| / k < 4.5 from 0.5 on), the series' below, the mean's
        assert abs(float(r.kl) - float(k)) <= 12 * u * float(k), q_
        want = -float(k + x) / 7  # dk/dlogp, of one token of seven
        assert (r.grad.double() + (-want)).abs().max() <= (8 * u + e) * abs(want), q_


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lengths", ["short", "many", "wide"])
def test_policy_terms_have_64_bits(lengths, dtype):
    """A gradient of 32 bits is off by its own rounding, of 2^-24, and 2^-32 of what it is made of: the ratio and the KL term alone too,
    as where a group's advantages are 0."""
    t, u = DT[dtype], 2.0 ** -24
    lp, old, off, mask, spans, keep = ragged(LENGTHS[lengths], t, 40, masked=0.2)
    gen = torch.Generator().manual_seed(4)
    ref = (torch.nan_to_num(lp.float().cpu(), nan=0.0) + 0.3 * torch.randn(lp.shape, generator=gen)).to(t).cuda()
    adv = torch.randn(len(spans), 1, generator=gen).to(t).cuda()
    tokens = torch.randn(lp.shape, generator=gen).to(t).cuda()
    for a, kl_coef, reduction in ((0 * adv, 0.1, "tokens"), (0 * tokens, 0.1, "tokens"), (0 * adv, 1.0, "sequences"), (adv, 0.0, "tokens"), (tokens, 0.0, "tokens"), (tokens, 0.3, "sequences")):
        r = losses.policy(lp, old, a, ref_logps=ref, offsets=off, mask=mask, kl_coef=kl_coef, reduction=reduction, wide_grad=True)
        f, kl, clip, grad, parts, size, klsize, _ = policy_in_64_bits(lp, old, a, ref, spans, keep, 0.2, 0.2, kl_coef, reduction)
        what = (lengths, dtype, kl_coef, reduction)
        near(r.grad, grad, 1.01 * u * grad.abs() + 2.0 ** -32 * parts, what)
        near(r.f, f, 1.01 * u * f.abs() + 2.0 ** -32 * (size + klsize), what)
        near(r.kl, kl, 1.01 * u * kl.abs(), what)


@pytest.mark.parametrize("bits", [32, 64])
def test_bad_offsets_give_nan(bits):
    """Offsets are data of the device: bad ones are clamped to the tokens there are, and the loss says so."""
    lp = -torch.rand(5000).cuda()
    for off in ([0, 3000, 2000, 4000, 5000], [-7, 10, 20, 30, 40], [0, 10, 20, 30, 5001], [9000, 9001, 9002, 9003, 9004]):
        o = torch.tensor(off, dtype=torch.int32 if bits == 32 else torch.int64).cuda()
        r = losses.preference(lp, offsets=o)
        assert r.f.isnan() and r.grad.shape == lp.shape
        r = losses.policy(lp, lp, torch.ones(4, 1).cuda(), offsets=o)
        assert r.f.isnan() and r.grad.shape == lp.shape
    o = torch.tensor([0, 1000, 1000, 1001, 5000], dtype=torch.int32 if bits == 32 else torch.int64).cuda()
    assert losses.preference(lp, offsets=o).f.isfinite()


def test_losses_beyond_32_bits():
    """More than 2^31 tokens; the second sequence reaches over all of them."""
    n = 2 ** 31 + 4099
    x = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    x[2], x[-1], x[n - 5000] = 1.0, -2.0, -4.0
    off = torch.tensor([0, 5, n], device="cuda")
    r = losses.preference(x, offsets=off, beta=0.5)
    slope = -0.5 / (1 + math.exp(3.5))  # h = 0.5 (1 - (-6))
    assert abs(float(r.f) - math.log1p(math.exp(-3.5))) < 1e-8 and r.rewards.tolist() == [0.5, -3.0]
    want = torch.tensor([slope, -slope]).to(torch.bfloat16).cuda()
    assert (r.grad[:5] == want[0]).all() and bool((r.grad[5:] == want[1]).all())
    del r
    p = losses.policy(x, x, x, offsets=off)  # every ratio is 1: f = -mean A, the gradient -A / N
    assert abs(float(p.f) - 5.0 / n) < 1e-15 and float(p.clip_fraction) == 0
    assert bool((p.grad.count_nonzero() == 3).all()) and abs(float(p.grad[-1]) * n - 2.0) < 2 * 2.0 ** -8
    p = losses.policy(x, x, torch.tensor([[1.0], [2.0]], device="cuda").bfloat16(), offsets=off, reduction="sequences")
    assert abs(float(p.f) + 1.5) < 1e-6 and abs(float(p.grad[-1]) * (n - 5) + 1.0) < 2.0 ** -7 and abs(float(p.grad[0]) * 5 + 0.5) < 2.0 ** -8


def test_losses_take_strided_tensors():
    base = -torch.rand(6, 40, 2).cuda()
    lp, old = base[:, 1:, 0], base[:, :-1, 1]
    mask = (torch.rand(6, 78).cuda() > 0.3)[:, ::2]
    a = losses.preference(lp, old, mask=mask)
    b = losses.preference(lp.contiguous(), old.contiguous(), mask=mask.contiguous())
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    adv = torch.randn(6, 78).cuda()[:, ::2]
    a = losses.policy(lp, old, adv, mask=mask)
    b = losses.policy(lp.contiguous(), old.contiguous(), adv.contiguous(), mask=mask.contiguous())
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    flat = base.reshape(-1)[1:]  # 4-byte aligned
    off = torch.tensor([0, 100, 200, 300, 479]).cuda()
    a, b = losses.preference(flat, offsets=off), losses.preference(flat.clone(), offsets=off)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_losses_autograd():
    lp, old, off, mask, spans, keep = ragged([30, 50, 7, 0], torch.float32, 3, masked=0.2)
    x = lp.clone().requires_grad_()
    (3.0 * losses.preference_loss(x, old, offsets=off, mask=mask)).backward()
    assert torch.equal(x.grad, 3.0 * losses.preference(lp, old, offsets=off, mask=mask).grad)
    x.grad = None
    f = losses.policy_loss(x, old, torch.ones(4, 1).cuda(), offsets=off, mask=mask)
    f.backward()
    r = losses.policy(lp, old, torch.ones(4, 1).cuda(), offsets=off, mask=mask)
    assert torch.equal(x.grad, r.grad) and torch.equal(f.detach(), r.f)
    assert not losses.policy_loss(lp, old, torch.ones(4, 1).cuda(), offsets=off, mask=mask).requires_grad


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lengths", ["short", "chunk", "many", "ones", "wide", [70001, 60000, 3, 0, 90000, 8]])
def test_16_bit_gradients_are_rounded_once(lengths, dtype):
    """Slopes of 1/tokens and 1/(pairs length) are not rounded to 16 bits, where f16 has few steps for them or none, before what
    comes into the loss -- a loss scale -- multiplies them.  In 32 bits as a direct result, too."""
    t, up = DT[dtype], 65536.0
    u, e, small = unit(t)
    lp, old, off, mask, spans, keep = ragged(LENGTHS.get(lengths) if isinstance(lengths, str) else lengths, t, 30, masked=0.1)
    scale = torch.tensor(up, device="cuda")
    for strided in (False, True):  # (native, and the way through Python)
        x = torch.stack((lp, lp), 1)[:, 0] if strided else lp.clone()
        x.requires_grad_()
        beta = 0.1
        _, _, want, size = preference_in_64_bits(lp, old, spans, keep, beta, "logistic", 0.0, True)
        sums = beta * beta * 4e-15 * (1 + float(size))
        wide = losses.preference(x.detach(), old, offsets=off, mask=mask, beta=beta, normalize_lengths=True, wide_grad=True)
        assert wide.grad.dtype == torch.float32
        near(wide.grad, want, u * 1.01 * want.abs() + sums, "preference")
        losses.preference_loss(x, old, offsets=off, mask=mask, beta=beta, normalize_lengths=True).backward(scale)
        # a 32-bit slope, its product (a power of two) and one rounding to 16 bits
        near(x.grad, want * up, (e + u) * 1.01 * (want * up).abs() + sums * up + small, "preference_loss")
        for adv, reduction in ((torch.randn(lp.shape, generator=torch.Generator().manual_seed(1)).to(t).cuda(), "tokens"),
                               (torch.randn(len(spans), 1, generator=torch.Generator().manual_seed(2)).to(t).cuda(), "sequences")):
            _, _, _, want, parts, *_ = policy_in_64_bits(lp, old, adv, None, spans, keep, 0.2, 0.2, 0.0, reduction)
            wide = losses.policy(x.detach(), old, adv, offsets=off, mask=mask, reduction=reduction, wide_grad=True)
            assert wide.grad.dtype == torch.float32
            near(wide.grad, want, u * 1.01 * want.abs() + 8 * u * parts, "policy")
            x.grad = None
            losses.policy_loss(x, old, adv, offsets=off, mask=mask, reduction=reduction).backward(scale)
            near(x.grad, want * up, (e + u) * 1.01 * (want * up).abs() + 8 * u * parts * up + small, "policy_loss")


def test_a_wide_gradient_of_wide_data_is_the_same():
    lp, old, off, mask, _, _ = ragged(LENGTHS["short"], torch.float32, 3, masked=0.2)
    for t in (torch.float32, torch.float64):
        a, b = (losses.preference(lp.to(t), old.to(t), offsets=off, mask=mask, wide_grad=w) for w in (False, True))
        c, d = (losses.policy(lp.to(t), old.to(t), old.to(t), offsets=off, mask=mask, wide_grad=w) for w in (False, True))
        assert a.grad.dtype == b.grad.dtype == d.grad.dtype == t and torch.equal(a.grad, b.grad) and torch.equal(c.grad, d.grad)


def test_losses_gradient_against_differences():
    lp, old, off, mask, spans, keep = ragged([9, 4, 6, 5], torch.float64, 5, masked=0.2)
    adv = torch.randn(24, dtype=torch.float64, generator=torch.Generator().manual_seed(0)).cuda()
    ref = old + 0.1
    h = 2.0 ** -20
    for call in (lambda x: losses.preference(x, old, offsets=off, mask=mask, beta=0.7, label_smoothing=0.1),
                 lambda x: losses.preference(x, old, offsets=off, mask=mask, beta=0.7, kind="squared", normalize_lengths=True),
                 lambda x: losses.policy(x, old, adv, ref_logps=ref, offsets=off, mask=mask, clip_low=0.9, clip_high=9.0, kl_coef=0.3)):
        grad = call(lp).grad.cpu()
        for t in keep.nonzero().flatten().tolist()[::3]:
            up, down = lp.clone(), lp.clone()
            up[t] += h
            down[t] -= h
            slope = float(call(up).f - call(down).f) / (2 * h)
            assert abs(slope - float(grad[t])) <= 100 * h * h + 1e-15 * 20 / h


# ------------------------------------------------------------------------------------ streams, graphs, devices
def three(seed):
    x, y, _ = make((8, 40), 517, torch.float32, seed)
    ref = losses.token_logprobs(make((8, 40), 517, torch.float32, seed + 1)[0], y)
    mask = torch.rand(8, 40, generator=torch.Generator().manual_seed(seed)).cuda() > 0.2
    return x, y, ref, mask


def chain(x, y, ref, mask):
    """A step as it is used: log-probabilities, both losses on them, back to the logits."""
    lp, lse = losses.token_logprobs_with_lse(x, y)
    r = losses.preference(lp, ref, mask=mask)
    p = losses.policy(lp, ref, r.rewards.unsqueeze(1), ref_logps=ref, mask=mask, kl_coef=0.1, reduction="sequences")
    return lp, r.f, r.rewards, p.f, p.kl, p.clip_fraction, losses.token_logprobs_grad(x, y, lse, r.grad + p.grad)


def test_results_are_the_same_bits_every_time_and_on_other_streams():
    args = three(0)
    want = chain(*args)
    big = ragged(LENGTHS["wide"], torch.float32, 1)
    first = losses.preference(big[0], big[1], offsets=big[2])
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s in streams:  # calls in flight beside each other
            with torch.cuda.stream(s):
                got.append((chain(*args), losses.preference(big[0], big[1], offsets=big[2])))
        torch.cuda.synchronize()
        for c, r in got:
            assert all(torch.equal(a, b) for a, b in zip(c, want))
            assert torch.equal(r.f, first.f) and torch.equal(r.grad, first.grad)


def test_captured_and_replayed():
    x, y, ref, mask = three(0)
    lp, old, off, _, _, _ = ragged(LENGTHS["chunk"], torch.float32, 1)
    step = lambda: chain(x, y, ref, mask) + tuple(losses.policy(lp, old, torch.ones(6, 1, device="cuda"), offsets=off))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for k in range(4):
        x.copy_(three(k + 5)[0])
        lp.add_(-0.01)
        want = step()
        for g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        torch.ones(1000, device="cuda").sum()


def test_native_calls_and_the_way_through_python_agree(monkeypatch):
    """What the native calls decline goes through Python's checks and copies to the same kernels."""
    from rust_lbfgs_amd import _train, directions

    lp, other, off, mask, _, _ = ragged([5, 0, 1, 17, 3, 2], torch.float32, 3, "packed", 0.3)
    x, y, g = make((3, 4), 1000, torch.bfloat16)
    w = torch.randn(3, 30, 50, generator=torch.Generator().manual_seed(1)).cuda()
    A = torch.randn(6, 1, generator=torch.Generator().manual_seed(2)).cuda()

    def everything():
        out = list(losses.token_logprobs_with_lse(x, y, 0.7, -1))
        out.append(losses.token_logprobs_grad(x, y, out[1], g, 0.7, -1))
        out += losses.preference(lp, other, offsets=off, mask=mask, beta=0.2, kind="squared", normalize_lengths=True)
        out += losses.policy(lp, other, A, ref_logps=other, offsets=off.int(), mask=mask, clip_low=0.1, clip_high=math.inf, kl_coef=0.1, reduction="sequences")
        out += losses.policy(lp.half().view(1, -1), other.half().view(1, -1), lp.half().view(1, -1), mask=mask.view(1, -1))
        return out + [directions.orthogonalize(w, steps=4, coefficients=(2, -1.5, 0.5))]

    native = everything()
    real = _train.calls()
    names = [n for n in dir(real) if not n.startswith("_")]
    declined = type("Declined", (), {n: staticmethod(lambda *a: None) for n in names})
    asked = []
    counting = type("Counting", (), {n: staticmethod(lambda *a, n=n: (asked.append(n), getattr(real, n)(*a))[1]) for n in names})
    monkeypatch.setattr(_train, "_CALLS", counting)
    done = everything()
    assert asked == ["logprobs", "logprobs_grad", "preference", "policy", "policy", "orthogonalize"]
    monkeypatch.setattr(_train, "_CALLS", declined)
    for a, b, c in zip(native, done, everything()):
        assert a.dtype == c.dtype and a.shape == c.shape and torch.equal(a.nan_to_num(7.0), c.nan_to_num(7.0)) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


def test_no_memory_is_torchs_own_error():
    x = torch.zeros(1 << 20, 65, dtype=torch.bfloat16, device="cuda")
    before = torch.cuda.memory_allocated()
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (64 << 20)) / torch.cuda.get_device_properties(0).total_memory)
    try:
        from rust_lbfgs_amd import directions

        with pytest.raises(torch.OutOfMemoryError):
            directions.orthogonalize(x)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert torch.cuda.memory_allocated() == before and losses.preference(torch.zeros(2, 3, device="cuda")).f.isfinite()


def test_autograd_forms_refuse_a_capture():
    x, y, ref, mask = three(0)
    x.requires_grad_()
    lp = torch.zeros(2, 4, device="cuda", requires_grad=True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for call in (lambda: losses.token_logprobs(x, y), lambda: losses.preference_loss(lp), lambda: losses.policy_loss(lp, lp.detach(), lp.detach())):
            with pytest.raises(RuntimeError, match="cannot be captured"):
                call()
        with torch.no_grad():
            out = losses.token_logprobs(x, y)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, losses.token_logprobs(x.detach(), y))


def test_tensors_on_different_devices_are_refused():
    lp = torch.zeros(2, 4, device="cuda")
    with pytest.raises(ValueError, match="is on"):
        losses.preference(lp, mask=torch.ones(2, 4, dtype=torch.bool))
    with pytest.raises(ValueError, match="is on"):
        losses.token_logprobs(lp, torch.zeros(2, dtype=torch.int64))


def test_forward_mode_derivatives_are_refused():
    """Dense plain tensors of the GPU, which the native calls would take, with a tangent that the result would not have."""
    from torch.autograd import forward_ad

    from rust_lbfgs_amd import directions

    x, y, g = make((3, 4), 50, torch.float32)
    lp = -torch.rand(4, 5).cuda()
    A = torch.ones(4, 1).cuda()
    _, lse = losses.token_logprobs_with_lse(x, y)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: losses.token_logprobs(dual(x), y), lambda: losses.token_logprobs(dual(x)[:, 1:], y[:, 1:]), lambda: losses.token_logprobs_with_lse(dual(x), y),
                     lambda: losses.token_logprobs_grad(dual(x), y, lse, g), lambda: losses.token_logprobs_grad(x, y, dual(lse), g),
                     lambda: losses.token_logprobs_grad(x, y, lse, dual(g)), lambda: losses.preference(dual(lp)), lambda: losses.preference_loss(lp, dual(lp)),
                     lambda: losses.policy(dual(lp), lp, lp), lambda: losses.policy_loss(lp, dual(lp), lp), lambda: losses.policy(lp, lp, dual(A)),
                     lambda: losses.policy(lp, lp, lp, ref_logps=dual(lp), kl_coef=0.1), lambda: directions.orthogonalize(dual(x[0]))):
            with pytest.raises(TypeError, match="forward-mode derivative"):
                call()
        assert losses.preference(lp).f.isfinite()  # a level alone takes nothing away


@pytest.mark.parametrize("bad", [dict(beta=-1.0), dict(label_smoothing=0.7), dict(label_smoothing=0.1, kind="hinge")])
def test_refused_calls_raise_and_leave_the_next_one_alone(bad):
    lp = -torch.rand(4, 5).cuda()
    with pytest.raises(LbfgsError):
        losses.preference(lp, **bad)
    assert losses.preference(lp).f.isfinite()


# ------------------------------------------------------------------------------------ together, under the optimiser
def test_the_optimiser_minimises_a_preference_loss():
    """x = an output projection in 64 bits; f and g through logits, token log-probabilities and the paired loss."""
    gen = torch.Generator().manual_seed(4)
    S, L, H, V = 8, 12, 10, 31
    hidden = torch.randn(S * L, H, dtype=torch.float64, generator=gen).cuda()
    tokens = torch.randint(0, V, (S, L), generator=gen).cuda()
    mask = (torch.arange(L)[None] < torch.tensor([12, 7, 1, 0, 12, 3, 5, 9])[:, None]).cuda()
    ref = torch.full((S, L), -math.log(V), dtype=torch.float64).cuda()

    def value_and_gradient(W):
        logits = (hidden @ W.t()).view(S, L, V)
        lp, lse = losses.token_logprobs_with_lse(logits, tokens)
        r = losses.preference(lp, ref, mask=mask, beta=0.5)
        dW = losses.token_logprobs_grad(logits, tokens, lse, r.grad).view(-1, V).t().contiguous() @ hidden
        return r.f + 0.05 * W.square().sum(), dW + 0.1 * W

    def evaluate(x, g):
        f, dW = value_and_gradient(x.view(V, H))
        g.copy_(dW.reshape(-1))
        return f

    W = torch.randn(V, H, dtype=torch.float64, generator=gen).cuda() * 0.1
    _, dW = value_and_gradient(W)
    D = torch.randn(V, H, dtype=torch.float64, generator=gen).cuda()
    h = 2.0 ** -18
    slope = float(value_and_gradient(W + h * D)[0] - value_and_gradient(W - h * D)[0]) / (2 * h)
    assert abs(slope - float((dW * D).sum())) <= 1e-7
    w = torch.nn.Parameter(W.clone())
    logits = (hidden @ w.t()).view(S, L, V)
    (losses.preference_loss(losses.token_logprobs(logits, tokens), ref, mask=mask, beta=0.5) + 0.05 * w.square().sum()).backward()
    assert (w.grad - dW).abs().max() <= 1e-14
    x = W.reshape(-1).cpu().numpy().copy()
    report = lbfgs().with_max_iterations(6).minimize(x, TorchEvaluate(evaluate))
    assert math.isfinite(report.fx) and abs(report.fx - float(value_and_gradient(torch.tensor(x).cuda().view(V, H))[0])) <= 1e-12
