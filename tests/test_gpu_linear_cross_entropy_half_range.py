"""linear_cross_entropy's gradients in half where 1 + 2 z lse is large: the gradient of the logits is kept times a power of two that leaves it within the type's range, so the
results are as exact, against float64, as elsewhere."""
import pytest
import torch

import catccos_amd as cc
from bounds16 import check, rounded, sum_error
from test_gpu_linear_cross_entropy import EXP

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[-1, 0, 1], ids=["chosen", "128x128", "256x256"], autouse=True)
def kernel16(request):
    """The kernel that a product goes to by itself, and each one that the loss has."""
    cc.set_option("matmul16_kernel", request.param)
    yield
    cc.set_option("matmul16_kernel", -1)


def _case(t, h, v, sure, below, seed=21):
    """Half of the tokens are up to `sure` certain of their target, half of another column; `below`: what is taken off every logit."""
    gen = torch.Generator().manual_seed(seed)
    w = torch.randn(v, h, generator=gen) * h ** -0.5
    tg = torch.randint(v, (t,), generator=gen)
    of = torch.where(torch.rand(t, generator=gen) < 0.5, tg, torch.randint(v, (t,), generator=gen))
    x = torch.randn(t, h, generator=gen) + sure * torch.rand(t, 1, generator=gen) * w[of]
    w[:, 0], x[:, 0] = -1.0, below
    tg[torch.rand(t, generator=gen) < 0.2] = -100
    return x.half(), w.half(), tg


def _kept_scale(most):
    """The largest power of two up to 2^11 that takes the largest value to 31 * 2^11 at most."""
    scale = 2.0 ** 11
    while most * scale > 31 * 2.0 ** 11:
        scale /= 2
    return scale


def _verify(t, h, v, z, sure, below, grad):
    x, w, tg = _case(t, h, v, sure, below)
    loss, nll, lse, tokens = cc.linear_cross_entropy(x.cuda(), w.cuda(), tg.cuda(), z_coef=z)
    got = cc.linear_cross_entropy_backward(torch.full((), grad, device="cuda"), x.cuda(), w.cuda(), tg.cuda(), lse, tokens, z_coef=z)
    use = tg >= 0
    n = int(use.sum())
    xd, wd, at = x[use].double(), w.double(), tg[use]
    l = xd @ wd.t()
    el = sum_error(xd, wd.t())
    s = torch.logsumexp(l, 1)
    es = el.amax(1) + EXP + (128 + v / 4096) * 2.0 ** -24 + 2.0 ** -22 * s.abs()
    f = (1 + 2 * z * s)[:, None]
    p = torch.exp(l - s[:, None])
    d = p * f
    d[torch.arange(n), at] -= 1
    most = float(torch.maximum(f.abs(), (1 - f).abs()).max())
    assert most > 32
    # p is off by its exponent's error and the hardware exponential's, f by lse's and two roundings; then d is rounded, its smallest step 2^-25 divided by what it is kept times
    ed = p * f.abs() * (2 * (el + es[:, None]) + EXP + 2.0 ** -22) + p * 2 * abs(z) * es[:, None] + 2.0 ** -23 * d.abs()
    ed = ed + torch.finfo(torch.float16).eps / 2 * (d.abs() + ed) + 2.0 ** -25 / _kept_scale(most)
    c = grad / n
    for name, g, a, b, ea in (("grad_x", got[0][use.cuda()], d, wd, ed), ("grad_w", got[1], d.t(), xd, ed.t())):
        y = a @ b * c
        assert float(y.abs().max()) < 60000
        check(g, y, rounded(y, (ea @ b.abs() + sum_error(a.abs() + ea, b) * 2) * c + 2.0 ** -22 * y.abs(), torch.float16), name)
    assert not got[0][~use.cuda()].any()
    # through autograd: the same bits
    xr, wr = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    (cc.linear_cross_entropy(xr, wr, tg.cuda(), z_coef=z)[0] * grad).backward()
    assert torch.equal(xr.grad, got[0]) and torch.equal(wr.grad, got[1])


@pytest.mark.parametrize("t,h,v,z,sure,below,grad", [
    (70, 64, 200, 0.5, 60.0, 0.0, 16.0),        # 1 + 2 z lse about 60
    (300, 136, 1000, 2.0, 50.0, 0.0, 4.0),      # 200
    (257, 77, 333, 1.0, 5.0, 40.0, 16.0),       # -70: all logits lie far below zero
    (40, 64, 130, -0.5, 60.0, 0.0, 16.0),       # -60
    (130, 72, 520, 1e3, 60.0, 0.0, 2.0 ** -6),  # 10^5, past what half holds at all
    (1000, 64, 4100, 0.3, 70.0, 0.0, 64.0)])
def test_gradients(t, h, v, z, sure, below, grad):
    _verify(t, h, v, z, sure, below, grad)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_token_that_is_not_finite_leaves_the_others_alone(bad):
    """What a NaN or infinite token's lse says of the range counts for nothing: the other tokens' rows are those without it."""
    x, w, tg = _case(60, 64, 200, 60.0, 0.0)
    tg = tg.clamp_min(0)
    x[7] = bad
    keep = torch.arange(60) != 7
    one = torch.full((), 0.25, device="cuda")
    grads = []
    for xs, ts in ((x, tg), (x[keep], tg[keep])):
        _, _, lse, tokens = cc.linear_cross_entropy(xs.cuda(), w.cuda(), ts.cuda(), reduction="sum", z_coef=1.0)
        grads.append(cc.linear_cross_entropy_backward(one, xs.cuda(), w.cuda(), ts.cuda(), lse, tokens, reduction="sum", z_coef=1.0)[0])
    assert torch.equal(grads[0][keep.cuda()], grads[1]) and bool(torch.isfinite(grads[1]).all()) and bool(torch.isnan(grads[0][7]).all())


def test_a_vocabulary_of_several_pieces():
    """Every piece of the vocabulary, and the sums over them, take the one scale."""
    _verify(66000, 24, 3700, 0.5, 60.0, 0.0, 1024.0)


def test_a_recorded_step_follows_the_range():
    """The scale is chosen on the device: a replay on values of another range equals the eager calls on them."""
    x, w, tg = (v.cuda() for v in _case(130, 72, 520, 60.0, 0.0))
    one = torch.full((), 0.25, device="cuda")

    def step():
        out = cc.linear_cross_entropy(x, w, tg, z_coef=2.0)
        return out + cc.linear_cross_entropy_backward(one, x, w, tg, out[2], out[3], z_coef=2.0)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for factor in (1.0, 0.03, 4.0, 1.0):
        x.copy_(_case(130, 72, 520, 60.0, 0.0)[0].cuda() * factor)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step())) and bool(torch.isfinite(held[4]).all())
