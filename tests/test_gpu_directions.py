"""Orthogonalised updates on the GPU against their definition in 64 bits.

The tolerance follows the errors through the steps: what is rounded away before the last j steps, relative to |X|_F, is
multiplied by at most the Lipschitz constant of the remaining map of the singular values (an odd function f acts on a matrix's
singular values with the constant max |f'| in the Frobenius norm).  A step rounds S, P and X to 22 bits (2^-23 each, S and P
acting through P's own size: counted 4 times) and accumulates in 32.  Of 16-bit updates of a short side beyond 64 the last g
steps are on the Gram matrix, where a rounding of 2^-23 becomes |b| a^(2 g - 2) 2^-23 of the result: g = 4 for bf16 and 3 for f16
with the usual polynomial, and as many as keep that below 2^-10 and 2^-13 with any."""
import math

import pytest
import torch

from rust_lbfgs_amd import LbfgsError, directions

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ABC = directions.COEFFICIENTS


def in_64_bits(g, steps, abc, device="cpu"):
    x = g.double().to(device)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    n = x.square().sum((-2, -1), keepdim=True).sqrt()
    x = torch.where(n > 0, x / n, 0.0)
    a, b, c = abc
    trail = [x]
    for _ in range(steps):
        s = x @ x.mT
        x = a * x + (b * s + c * (s @ s)) @ x
        trail.append(x)
    return (x.mT if tall else x), trail


def tolerance(g, trail, abc, dtype):
    """Relative to the result, in the Frobenius norm, of the worst matrix of the batch."""
    a, b, c = abc
    worst = 0.0
    flat = [t.reshape(-1, *t.shape[-2:]) for t in trail]
    for k in range(flat[0].shape[0]):
        norms = [float(t[k].norm()) for t in flat]
        if not math.isfinite(norms[-1]) or norms[-1] == 0:
            continue
        off = 0.0
        for j in range(len(flat)):
            top = float(torch.linalg.matrix_norm(flat[j][k], 2)) if min(flat[j][k].shape) else 0.0
            s = torch.linspace(0, top * 1.001 + 1e-12, 4001, dtype=torch.float64)
            slope = torch.ones_like(s)
            for _ in range(len(flat) - 1 - j):
                slope = slope * (a + 3 * b * s ** 2 + 5 * c * s ** 4)
                s = a * s + b * s ** 3 + c * s ** 5
            scale = max(1.0, abs(a)) if j else 1.0
            off += float(slope.abs().max()) * 12 * 2.0 ** -23 * scale * norms[j]
        worst = max(worst, off / norms[-1])
    return worst + torch.finfo(dtype).eps / 2 + (on_the_gram_matrix(dtype) if min(g.shape[-2:]) > 64 or len(flat) > 8 else 0)


def on_the_gram_matrix(dtype):
    return {torch.float32: 0.0, torch.bfloat16: 2.0 ** -10, torch.float16: 2.0 ** -13}[dtype]


def check_large(g, steps=5):
    """The same in the Frobenius norm of the whole, with the 64-bit products on the GPU and the errors' growth from the power
    iteration's bound on |X| (singular values of [0, 1.21] are within the polynomial's range): a^(steps left), at most."""
    got = directions.orthogonalize(g, steps=steps).double()
    flat = g.reshape(-1, *g.shape[-2:])
    for k, x in enumerate(got.reshape(flat.shape)):
        want, trail = in_64_bits(flat[k], steps, ABC, "cuda")
        norms = [float(t.norm()) for t in trail]
        off = sum(ABC[0] ** (steps - j) * 12 * 2.0 ** -23 * ABC[0] * norms[j] for j in range(steps + 1)) / norms[-1]
        off += on_the_gram_matrix(g.dtype)
        assert float((x - want).norm()) <= (off + torch.finfo(g.dtype).eps / 2) * norms[-1], (k, float((x - want).norm()) / norms[-1], off)
        # and nowhere far off: no block of the result is another's
        assert float((x - want).abs().max()) <= 40 * (off + torch.finfo(g.dtype).eps / 2) * max(norms[-1] / want.numel() ** 0.5, float(want.abs().max()) / 8)


def check(g, steps=5, abc=ABC):
    before = g.clone()
    got = directions.orthogonalize(g, steps=steps, coefficients=abc)
    assert torch.equal(g, before) and got.shape == g.shape and got.dtype == g.dtype and got.is_contiguous()
    want, trail = in_64_bits(g, steps, abc)
    tol = tolerance(g, trail, abc, g.dtype)
    x, y = got.double().cpu().reshape(-1, *g.shape[-2:]), want.reshape(-1, *g.shape[-2:])
    for k in range(x.shape[0]):
        n = float(y[k].norm())
        assert float((x[k] - y[k]).norm()) <= tol * n, (k, float((x[k] - y[k]).norm()) / n, tol)
    return got, want


def gradient(*shape, dtype=torch.float32, seed=0, rank=8, noise=0.3):
    gen = torch.Generator().manual_seed(seed)
    lead, (m, n) = shape[:-2], shape[-2:]
    g = torch.randn(*lead, m, rank, generator=gen) @ torch.randn(*lead, rank, n, generator=gen) / math.sqrt(rank) + noise * torch.randn(*shape, generator=gen)
    return g.to(dtype).cuda()


SIZES = [(1, 1), (1, 9), (9, 1), (2, 3), (16, 16), (31, 33), (64, 64), (65, 63), (100, 300), (128, 128), (129, 127), (300, 128), (256, 512), (400, 401), (333, 1000)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m, n", SIZES)
def test_sizes(m, n, dtype):
    check(gradient(m, n, dtype=DT[dtype]))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape", [(3, 40, 50), (2, 3, 130, 70), (5, 200, 600), (1, 1, 20, 20), (17, 8, 8)])
def test_batches(shape, dtype):
    g = gradient(*shape, dtype=DT[dtype])
    got, _ = check(g)
    one = directions.orthogonalize(g.reshape(-1, *shape[-2:])[1 if g.numel() > shape[-1] * shape[-2] else 0])
    assert torch.equal(one, got.reshape(-1, *shape[-2:])[1 if g.numel() > shape[-1] * shape[-2] else 0])  # a matrix is what it is alone


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape", [(700, 900), (1500, 500), (512, 2100), (1030, 1030)])
def test_larger(shape, dtype):
    check(gradient(*shape, dtype=DT[dtype], rank=32))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape", [(2100, 2300), (4000, 4100), (1100, 8200), (4, 1024, 2048), (3, 1500, 700), (12, 520, 600), (40, 260, 300)])
def test_every_tile(shape, dtype):
    """Sizes at which products go by tiles of 64, 128 (one and two to a unit) and 192, single and paired."""
    check_large(gradient(*shape, dtype=DT[dtype], rank=64))


def check_short(g, steps=5, abc=ABC):
    """A short side up to 64: all in 64 bits, so that the result is the definition's rounded once, and as much as 2^-26 beside
    (a rounding of 2^-52 times the steps' growth |b| a^(2 steps - 2), where that is what decides for 64 bits)."""
    got = directions.orthogonalize(g, steps=steps, coefficients=abc)
    want, _ = in_64_bits(g, steps, abc)
    x, info = got.double().cpu(), torch.finfo(g.dtype)
    beside = 2.0 ** -26 * want.square().sum((-2, -1), keepdim=True).sqrt()
    assert got.shape == g.shape and got.dtype == g.dtype
    assert ((x - want).abs() <= (want.abs() + beside) * (info.eps / 2) + info.smallest_normal * info.eps / 2 + beside).all()
    return got


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape", [(1, 1), (1, 100000), (7, 3), (15, 16), (16, 64), (17, 65), (32, 31), (33, 4097), (47, 48), (49, 1000), (63, 5000), (64, 64), (64, 8191), (2000, 64), (777, 31), (70001, 2), (5000, 48)])
def test_a_short_side(shape, dtype):
    check_short(gradient(*shape, dtype=DT[dtype]))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape", [(1100, 5, 9), (300, 33, 130), (2, 700, 20, 11), (40, 64, 1300), (5000, 1, 3)])
def test_batches_of_a_short_side(shape, dtype):
    got = check_short(gradient(*shape, dtype=DT[dtype]))
    assert torch.equal(got, directions.orthogonalize(gradient(*shape, dtype=DT[dtype])))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("steps, abc", [(1, ABC), (2, ABC), (3, ABC), (6, ABC), (7, ABC), (20, (1.5, -0.5, 0.0)), (4, (15 / 8, -10 / 8, 3 / 8)), (2, (-1.0, 0.0, 0.5)), (1, (1.0, 0.0, 0.0)), (3, (0.0, 0.0, 0.0))])
def test_steps_and_coefficients_of_a_short_side(steps, abc, dtype):
    check_short(gradient(40, 300, dtype=DT[dtype]), steps, abc)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("steps, abc", [(8, ABC), (30, (1.5, -0.5, 0.0))])
def test_more_steps_of_a_short_side_than_64_bits_have_room_for(steps, abc, dtype):
    check(gradient(40, 300, dtype=DT[dtype], rank=40), steps, abc)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape", [(65, 65), (65, 1000), (96, 97), (96, 1536), (96, 1537), (97, 512), (128, 129), (128, 513), (128, 768), (128, 769), (4096, 128), (4097, 100), (700, 66),
                                   (30, 100, 500), (20, 70, 260), (2, 128, 130, 90), (300, 80, 90)])
def test_a_side_of_up_to_128(shape, dtype):
    """One launch a step, panels of 64 and 128 columns, and where that ends."""
    g = gradient(*shape, dtype=DT[dtype])
    got, _ = check(g) if g.numel() < 400000 else (directions.orthogonalize(g), check_large(g))
    assert torch.equal(got, directions.orthogonalize(g))


@pytest.mark.parametrize("dtype", DT)
def test_bad_values_of_a_side_of_up_to_128_stay_with_their_matrix(dtype):
    g = gradient(5, 130, 75, dtype=DT[dtype])
    g[1] = 0
    g[2, 129, 74] = math.nan
    g[3, 0, 0] = -math.inf
    got = directions.orthogonalize(g)
    assert (got[1] == 0).all() and got[2].isnan().all() and got[3].isnan().all()
    for k in (0, 4):
        assert torch.equal(got[k], directions.orthogonalize(g[k]))
        assert torch.equal(got[k].t(), directions.orthogonalize(g[k].t().contiguous()))


def test_many_steps_of_a_short_side_and_no_full_rank():
    for shape in ((40, 300), (64, 64), (300, 20)):
        for dtype in DT.values():
            for steps in (7, 8, 12, 64):  # (what is zero but for roundings may have grown to one, and stays there)
                got = directions.orthogonalize(gradient(*shape, dtype=dtype, rank=3, noise=0.0), steps=steps).double()
                assert got.isfinite().all() and float(torch.linalg.matrix_norm(got.cpu(), 2)) < 1.4


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape", [(90, 140), (40, 70)])
def test_a_steep_polynomial(shape, dtype):
    """The growth of errors on the Gram matrix, and with it the number of steps there, depends on the polynomial: with Chebyshev's of
    degree 5, of [0, 1] into [-1, 1] at slopes up to 25, two of three steps for bf16, one for f16, all five for a short side."""
    t5 = (5.0, -20.0, 16.0)
    check(gradient(*shape, dtype=DT[dtype], rank=90), 3, t5)
    if min(shape) <= 64:
        check_short(gradient(*shape, dtype=DT[dtype], rank=90), 5, t5)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("steps, abc", [(1, ABC), (2, ABC), (6, ABC), (8, (1.5, -0.5, 0.0)), (4, (15 / 8, -10 / 8, 3 / 8)), (3, (0.0, 0.0, 0.0)), (2, (-1.0, 0.0, 0.5)), (1, (1.0, 0.0, 0.0))])
def test_steps_and_coefficients(steps, abc, dtype):
    g = gradient(90, 140, dtype=DT[dtype])
    got, want = check(g, steps, abc) if abc != (0.0, 0.0, 0.0) else (directions.orthogonalize(g, steps=steps, coefficients=abc), None)
    if want is None:
        assert (got == 0).all()


@pytest.mark.parametrize("shape", [(60, 100), (200, 150), (256, 2000)])
def test_low_rank_and_ill_conditioned(shape):
    for dtype in DT.values():
        check(gradient(*shape, dtype=dtype, rank=1, noise=0.0))
        check(gradient(*shape, dtype=dtype, rank=4, noise=1e-3))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rank, noise", [(4, 1e-3), (4, 1e-4), (32, 1e-3)])
@pytest.mark.parametrize("shape", [(256, 2000), (200, 150), (512, 4000)])
def test_little_is_lost_beside_the_rounding_of_the_result(shape, rank, noise, dtype):
    """Of 16-bit updates nearly without noise: a difference between the halves of a symmetric matrix, or a value whose two parts do
    not fit each other, would be multiplied by up to a^2 in every step.  Over 30000 elements and more, the rounding of the result and
    that of the definition's are alike in their norm to some 1/sqrt(30000) < 5 %."""
    g = gradient(*shape, dtype=DT[dtype], rank=rank, noise=noise)
    want, _ = in_64_bits(g, 5, ABC, "cuda")
    rounding, n = float((want.to(g.dtype).double() - want).norm()), float(want.norm())
    assert float((directions.orthogonalize(g).double() - want).norm()) <= 1.05 * rounding + on_the_gram_matrix(g.dtype) * n


@pytest.mark.parametrize("dtype", DT)
def test_the_scale_of_an_update_does_not_matter(dtype):
    t = DT[dtype]
    g = gradient(70, 110, dtype=t)
    want = directions.orthogonalize(g)
    for k in (-12, 9) if t == torch.float16 else (-120, -60, 90):
        h = g * 2.0 ** k
        if torch.equal(h.double() * 2.0 ** -k, g.double()):
            assert torch.equal(directions.orthogonalize(h), want), k
        else:  # entries below the type's smallest normal number lost bits: another matrix
            check(h)


@pytest.mark.parametrize("dtype", DT)
def test_zeros_and_bad_values_stay_with_their_matrix(dtype):
    g = gradient(5, 60, 80, dtype=DT[dtype])
    g[1] = 0
    g[2, 3, 4] = math.nan
    g[3, 0, 0] = math.inf
    got = directions.orthogonalize(g)
    assert (got[1] == 0).all() and got[2].isnan().all() and got[3].isnan().all()
    for k in (0, 4):
        assert torch.equal(got[k], directions.orthogonalize(g[k]))
    assert directions.orthogonalize(torch.zeros(0, 3, 4, device="cuda")).shape == (0, 3, 4)
    assert directions.orthogonalize(torch.zeros(3, 0, device="cuda")).shape == (3, 0)


def test_strided_updates():
    g = gradient(64, 200)
    assert torch.equal(directions.orthogonalize(g[:, ::2]), directions.orthogonalize(g[:, ::2].contiguous()))
    assert torch.equal(directions.orthogonalize(g.t()), directions.orthogonalize(g.t().contiguous()))
    base = torch.zeros(64 * 100 + 1, device="cuda")
    view = base[1:].view(64, 100)  # 4-byte aligned
    view.copy_(g[:, :100])
    assert torch.equal(directions.orthogonalize(view), directions.orthogonalize(g[:, :100].contiguous()))


def test_a_tall_update_is_the_wide_ones_transpose():
    for dtype in DT.values():
        g = gradient(130, 300, dtype=dtype)
        assert torch.equal(directions.orthogonalize(g.t().contiguous()), directions.orthogonalize(g).t())


def test_other_streams_and_two_calls_at_once():
    g, h = gradient(300, 500), gradient(4, 200, 200, dtype=torch.bfloat16)
    want = directions.orthogonalize(g), directions.orthogonalize(h)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append((directions.orthogonalize(g), directions.orthogonalize(h)))
        torch.cuda.synchronize()
        assert all(torch.equal(a, want[0]) and torch.equal(b, want[1]) for a, b in got)


def test_captured_and_replayed():
    g, h = gradient(100, 150), gradient(3, 260, 200, dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        directions.orthogonalize(g), directions.orthogonalize(h)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = directions.orthogonalize(g), directions.orthogonalize(h)
        graphs.append((graph, out))
    for k in range(4):
        g.copy_(gradient(100, 150, seed=k + 3))
        h.mul_(-1.5)
        want = directions.orthogonalize(g), directions.orthogonalize(h)
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        torch.ones(1000, device="cuda").sum()


def test_captured_and_replayed_with_short_sides():
    shapes = [(40, 700), (3, 64, 50), (100, 300), (2, 700, 90), (20, 9000)]
    g = [gradient(*shape, seed=k) for k, shape in enumerate(shapes)]
    for x in g:
        directions.orthogonalize(x)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = [directions.orthogonalize(x) for x in g]
        graphs.append((graph, out))
    for k in range(4):
        for n, x in enumerate(g):
            x.copy_(gradient(*shapes[n], seed=10 * k + n + 3))
        want = [directions.orthogonalize(x) for x in g]
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        torch.ones(1000, device="cuda").sum()


def test_refusals_raise():
    g = gradient(10, 10)
    with pytest.raises(LbfgsError, match="steps"):
        directions.orthogonalize(g, steps=0)
    with pytest.raises(LbfgsError, match="out of range"):
        directions.orthogonalize(g, coefficients=(5.0, 0.0, 0.0))
    assert directions.orthogonalize(g).isfinite().all()


def test_an_orthogonalised_descent_step():
    """A step as it is used: gradient of a loss, momentum, the direction, the parameter."""
    from rust_lbfgs_amd import losses

    gen = torch.Generator().manual_seed(0)
    W = torch.nn.Parameter((torch.randn(50, 24, generator=gen) * 0.1).cuda())
    hidden, y = torch.randn(64, 24, generator=gen).cuda(), torch.randint(0, 50, (4, 16), generator=gen).cuda()
    old = losses.token_logprobs((hidden @ W.detach().t()).view(4, 16, 50), y)
    adv = torch.randn(4, 1, generator=gen).cuda()
    momentum = torch.zeros_like(W)
    for _ in range(3):
        W.grad = None
        losses.policy_loss(losses.token_logprobs((hidden @ W.t()).view(4, 16, 50), y), old, adv).backward()
        momentum.mul_(0.9).add_(W.grad)
        d = directions.orthogonalize(momentum)
        want, trail = in_64_bits(momentum, 5, ABC)
        assert float((d.double().cpu() - want).norm()) <= tolerance(momentum, trail, ABC, d.dtype) * float(want.norm())
        with torch.no_grad():
            W.sub_(0.02 * d)
    assert W.isfinite().all()


def test_the_example_takes_the_optimisers_gradients():
    import re

    example = re.search(r"    d = (directions\.orthogonalize\(.*\))  ", directions.__doc__).group(1)
    g = torch.randn(30 * 50, dtype=torch.float64, generator=torch.Generator().manual_seed(0)).cuda()
    d = eval(example, dict(directions=directions, gradient=g, rows=30, cols=50))
    used = -g.view(30, 50).float()
    want, trail = in_64_bits(used, 5, ABC)
    assert d.dtype == torch.float32 and float((d.double().cpu() - want.cpu()).norm()) <= tolerance(used, trail, ABC, d.dtype) * float(want.norm())
