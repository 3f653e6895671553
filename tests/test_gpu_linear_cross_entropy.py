"""linear_cross_entropy and its gradients against float64, within bounds derived here and in bounds16.py."""
import pytest
import torch

import catccos_amd as cc
from bounds16 import check, rounded, sum_error

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[-1, 0, 1, 2], ids=["chosen", "128x128", "256x256", "rows"], autouse=True)
def kernel16(request):
    """The kernel that a product goes to by itself, and each one."""
    cc.set_option("matmul16_kernel", request.param)
    yield
    cc.set_option("matmul16_kernel", -1)

# The sum of a row's exponentials: each is off by a few units in the last place and by its argument's rounding, 2^-24 times an argument that matters up to about 40; a sum of
# 64 columns, then of their statistics over 64 lanes and along V / 4096 of them: fewer than 128 + V / 4096 additions deep.
EXP = 2.0 ** -18


def _case(t, h, v, dtype, ignored=0.3, seed=3, target=torch.int64):
    gen = torch.Generator().manual_seed(seed)
    w = (torch.randn(v, h, generator=gen) * h ** -0.5).to(dtype)
    tg = torch.randint(v, (t,), generator=gen)
    x = (torch.randn(t, h, generator=gen) + 8 * torch.rand(t, 1, generator=gen) * w[tg].float()).to(dtype)
    out = torch.rand(t, generator=gen) < ignored
    tg[out] = torch.tensor([-100, -1, v, v + 7])[torch.randint(4, (int(out.sum()),), generator=gen)]
    return x, w, tg.to(target)


def _verify(x, w, tg, got, grads=None, z=0.0, reduction="mean", scale=1.0):
    t, v = x.shape[0], w.shape[0]
    dtype = x.dtype
    use = (tg >= 0) & (tg < v)
    n = int(use.sum())
    xd, wd, at = x[use].double(), w.double(), tg[use].long()
    l = xd @ wd.t()
    el = sum_error(xd, wd.t())
    lse = torch.logsumexp(l, 1)
    elog = el.amax(1) if l.numel() else lse
    elog = elog + EXP + (128 + v / 4096) * 2.0 ** -24 + 2.0 ** -22 * lse.abs()
    nll = lse - l.gather(1, at[:, None]).squeeze(1)
    enll = elog + el.gather(1, at[:, None]).squeeze(1) + 2.0 ** -23 * nll.abs()

    def whole(a):
        o = torch.zeros((t,) + a.shape[1:], dtype=torch.float64)
        o[use] = a
        return o

    loss, g_nll, g_lse, tokens = got
    check(g_lse, whole(lse), whole(elog), "lse")
    check(g_nll, whole(nll), whole(enll), "nll")
    assert tokens.tolist() == [n] and tokens.dtype == torch.int32
    share = 1.0 if reduction == "sum" else 1.0 / max(n, 1)
    want = ((nll + z * lse * lse) * share).sum()
    tol = ((enll + 2 * z * lse.abs() * elog) * share).sum() + 2.0 ** -22 * want.abs() + 1e-30
    check(loss.reshape(1), want.reshape(1), tol.reshape(1), "loss")
    if grads is None:
        return
    p = torch.exp(l - lse[:, None])
    f = (1 + 2 * z * lse)[:, None]
    d = p * f
    d[torch.arange(n), at] -= 1
    # p is off by its exponent's error and the hardware exponential's, then d is rounded (half: times 2^11, so that its smallest step is 2^-25 / 2^11)
    ed = p * f * (2 * (el + elog[:, None]) + EXP) + 2.0 ** -23 * d.abs()
    ed = ed + torch.finfo(dtype).eps / 2 * (d.abs() + ed) + (2.0 ** -36 if dtype == torch.float16 else 0.0)
    c = share * scale
    for name, g, a, b, ea in (("grad_x", grads[0], d, wd, ed), ("grad_w", grads[1], d.t(), xd, ed.t())):
        if g is None:
            continue
        y = a @ b * c
        e = (ea @ b.abs() + sum_error(a.abs() + ea, b) * 2) * c + 2.0 ** -22 * y.abs()
        b16 = rounded(y, e, dtype)
        check(g, whole(y) if name == "grad_x" else y, whole(b16) if name == "grad_x" else b16, name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,h,v,ignored,z,reduction", [
    (1, 64, 64, 0.0, 0.0, "mean"), (1, 8, 1, 0.0, 0.0, "mean"), (5, 72, 100, 0.4, 1e-3, "sum"), (64, 256, 1000, 0.0, 0.0, "mean"), (130, 136, 520, 0.5, 1e-4, "mean"),
    (300, 77, 333, 0.3, 0.0, "mean"), (257, 512, 2049, 0.2, 1e-2, "sum"), (1000, 64, 4100, 0.7, 0.0, "mean"), (513, 200, 771, 0.0, 1e-4, "mean")])
def test_loss_and_gradients(t, h, v, ignored, z, reduction, dtype):
    x, w, tg = _case(t, h, v, dtype, ignored)
    scale = 1024.0 if dtype == torch.float16 else 1.0
    xd, wd, td = x.cuda(), w.cuda(), tg.cuda()
    got = cc.linear_cross_entropy(xd, wd, td, reduction=reduction, z_coef=z)
    grad = torch.full((), scale, device="cuda")
    grads = cc.linear_cross_entropy_backward(grad, xd, wd, td, got[2], got[3], reduction=reduction, z_coef=z)
    _verify(x, w, tg, got, grads, z, reduction, scale)
    xr, wr = xd.clone().requires_grad_(), wd.clone().requires_grad_()
    loss, nll, lse, tokens = cc.linear_cross_entropy(xr, wr, td.int(), reduction=reduction, z_coef=z)
    (loss * scale).backward()
    assert all(torch.equal(a, b) for a, b in zip((loss, nll, lse, tokens), got))
    assert torch.equal(xr.grad, grads[0]) and torch.equal(wr.grad, grads[1])
    assert not nll.requires_grad and not lse.requires_grad


@pytest.mark.parametrize("z", [0.0, 1e-2])
def test_against_differences(z):
    """In float64 around the same values: the gradient of the plain loss in a few directions, and this one's within what its roundings allow (a handful of eps / 2)."""
    x, w, tg = _case(24, 40, 90, torch.float16, 0.25, seed=8)
    xr, wr = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    (cc.linear_cross_entropy(xr, wr, tg.cuda(), z_coef=z)[0] * 4096).backward()
    use = (tg >= 0) & (tg < 90)

    def value(a, b):
        l = a[use] @ b.t()
        s = torch.logsumexp(l, 1)
        return (s - l.gather(1, tg[use][:, None]).squeeze(1) + z * s * s).mean()

    gen = torch.Generator().manual_seed(2)
    for leaf, which in ((xr, 0), (wr, 1)):
        base = [x.double(), w.double()]
        d = torch.randn(base[which].shape, generator=gen, dtype=torch.float64)
        hi, lo = list(base), list(base)
        hi[which], lo[which] = base[which] + 1e-5 * d, base[which] - 1e-5 * d
        diff = float((value(*hi) - value(*lo)) / 2e-5)
        got = leaf.grad.double().cpu() / 4096
        assert abs(float((got * d).sum()) - diff) <= 4 * torch.finfo(torch.float16).eps * float((got.abs() * d.abs()).sum()) + 1e-7


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tokens_that_do_not_count_hold_anything(dtype):
    x, w, tg = _case(200, 72, 300, dtype, 0.5)
    out = (tg < 0) | (tg >= 300)
    want = cc.linear_cross_entropy(x.cuda(), w.cuda(), tg.cuda(), z_coef=1e-3)
    one = torch.ones((), device="cuda")
    grads = cc.linear_cross_entropy_backward(one, x.cuda(), w.cuda(), tg.cuda(), want[2], want[3], z_coef=1e-3)
    x[out] = torch.tensor([float("nan"), float("inf"), -float("inf")])[torch.arange(int(out.sum())) % 3][:, None].to(dtype)
    got = cc.linear_cross_entropy(x.cuda(), w.cuda(), tg.cuda(), z_coef=1e-3)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    again = cc.linear_cross_entropy_backward(one, x.cuda(), w.cuda(), tg.cuda(), got[2], got[3], z_coef=1e-3)
    assert torch.equal(again[0], grads[0]) and torch.equal(again[1], grads[1])
    assert not again[0][out.cuda()].any()


@pytest.mark.parametrize("t", [0, 3])
def test_no_token_counts(t):
    x = torch.randn(t, 32, device="cuda").bfloat16().requires_grad_()
    w = torch.randn(50, 32, device="cuda").bfloat16().requires_grad_()
    loss, nll, lse, tokens = cc.linear_cross_entropy(x, w, torch.full((t,), -100, device="cuda"), z_coef=0.1)
    assert float(loss) == 0 and not nll.any() and not lse.any() and tokens.tolist() == [0]
    loss.backward()
    assert not x.grad.any() and not w.grad.any()


def test_a_mean_over_more_tokens():
    """tokens is what a mean divides by: twice as many halve the gradients (exactly, a power of two)."""
    x, w, tg = (v.cuda() for v in _case(64, 64, 200, torch.bfloat16, 0.0))
    _, _, lse, tokens = cc.linear_cross_entropy(x, w, tg)
    one = torch.ones((), device="cuda")
    a = cc.linear_cross_entropy_backward(one, x, w, tg, lse, tokens)
    b = cc.linear_cross_entropy_backward(one, x, w, tg, lse, tokens * 2)
    assert torch.equal(a[0], b[0] * 2) and torch.equal(a[1], b[1] * 2)


def test_a_token_that_is_not_finite_shows():
    x, w, tg = _case(40, 64, 200, torch.bfloat16, 0.0)
    x[7] = float("nan")
    loss, nll, lse, _ = cc.linear_cross_entropy(x.cuda(), w.cuda(), tg.cuda())
    assert torch.isnan(loss) and torch.isnan(nll[7]) and torch.isnan(lse[7])
    keep = torch.arange(40) != 7
    want = cc.linear_cross_entropy(x[keep].cuda(), w.cuda(), tg[keep].cuda())
    assert torch.equal(nll[keep.cuda()], want[1]) and torch.equal(lse[keep.cuda()], want[2])


def test_refusals():
    x, w, tg = (v.cuda() for v in _case(20, 16, 30, torch.bfloat16))
    loss, nll, lse, tokens = cc.linear_cross_entropy(x, w, tg)
    one = torch.ones((), device="cuda")
    for bad in (lambda: cc.linear_cross_entropy(x.float(), w, tg), lambda: cc.linear_cross_entropy(x, w.half(), tg), lambda: cc.linear_cross_entropy(x, w[:, :8], tg),
                lambda: cc.linear_cross_entropy(x, w, tg.short()), lambda: cc.linear_cross_entropy(x, w, tg[:3]), lambda: cc.linear_cross_entropy(x, w, tg, reduction="none"),
                lambda: cc.linear_cross_entropy(x, w.cpu(), tg), lambda: cc.linear_cross_entropy_backward(one.double(), x, w, tg, lse, tokens),
                lambda: cc.linear_cross_entropy_backward(one, x, w, tg, lse[:3], tokens), lambda: cc.linear_cross_entropy_backward(one, x, w, tg, lse, tokens.long())):
        with pytest.raises(ValueError):
            bad()
