"""grouped_matmul and its gradients against float64 products of the same 16-bit operands, within bounds derived in bounds16.py."""
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

SIZES = [
    # group sizes, rows behind the last group, k, n
    ([1], 0, 64, 64),
    ([5, 0, 3], 2, 64, 40),
    ([0, 0, 7, 0], 0, 24, 8),
    ([0, 0, 0], 9, 32, 16),
    ([300, 1, 0, 129, 128], 33, 192, 264),
    ([257, 511], 0, 1000, 520),
    ([31, 32, 33, 63, 64, 65], 1, 136, 72),
    ([17, 4], 3, 77, 33),          # rows of no whole 16 bytes
    ([2, 90], 0, 200, 131),
    ([40, 9], 1, 131, 256),
    ([700, 650], 50, 520, 768),
]


def _case(sizes, rest, k, n, trans_b, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    t, e = sum(sizes) + rest, len(sizes)
    x = torch.randn(t, k, generator=gen).to(dtype)
    w = (torch.randn(e, n, k, generator=gen) if trans_b else torch.randn(e, k, n, generator=gen)).to(dtype)
    g = torch.randn(t, n, generator=gen).to(dtype)
    return x, w, g, torch.tensor(sizes, dtype=torch.int32)


def _ranges(sizes, t):
    at = 0
    for s in sizes:
        s = min(max(s, 0), t - at)
        yield at, at + s
        at += s


def _verify(got, x, w, sizes, trans_b, g=None, grads=None):
    t, n = got.shape
    dtype = x.dtype
    xd, wd = x.double(), w.double()
    want, bound = torch.zeros(t, n, dtype=torch.float64), torch.zeros(t, n, dtype=torch.float64)
    if grads is not None:
        gd = g.double()
        wx, bx = torch.zeros_like(xd), torch.zeros_like(xd)
        ww, bw = torch.zeros_like(wd), torch.zeros_like(wd)
    for i, (a, b) in enumerate(_ranges(sizes, t)):
        if a == b:
            continue
        m = wd[i].t() if trans_b else wd[i]
        want[a:b] = xd[a:b] @ m
        bound[a:b] = rounded(want[a:b], sum_error(xd[a:b], m), dtype)
        if grads is not None:
            wx[a:b] = gd[a:b] @ m.t()
            bx[a:b] = rounded(wx[a:b], sum_error(gd[a:b], m.t()), dtype)
            p, q = (gd[a:b].t(), xd[a:b]) if trans_b else (xd[a:b].t(), gd[a:b])
            ww[i] = p @ q
            bw[i] = rounded(ww[i], sum_error(p, q), dtype)
    check(got, want, bound, "out")
    if grads is not None:
        check(grads[0], wx, bx, "grad_x")
        check(grads[1], ww, bw, "grad_w")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("trans_b", [0, 1])
@pytest.mark.parametrize("sizes,rest,k,n", SIZES)
def test_products_and_gradients(sizes, rest, k, n, trans_b, dtype):
    x, w, g, gs = _case(sizes, rest, k, n, trans_b, dtype)
    xd, wd, gd, sd = (v.cuda() for v in (x, w, g, gs))
    out = cc.grouped_matmul(xd, wd, sd, trans_b=trans_b)
    grads = cc.grouped_matmul_backward(gd, xd, wd, sd, trans_b=trans_b)
    assert out.dtype == dtype and grads[0].dtype == dtype and grads[1].dtype == dtype
    _verify(out, x, w, sizes, trans_b, g, grads)
    # through autograd: the same bits
    xr, wr = xd.clone().requires_grad_(), wd.clone().requires_grad_()
    y = cc.grouped_matmul(xr, wr, sd, trans_b=trans_b)
    y.backward(gd)
    assert torch.equal(y, out) and torch.equal(xr.grad, grads[0]) and torch.equal(wr.grad, grads[1])


@pytest.mark.parametrize("trans_b", [0, 1])
def test_sizes_that_do_not_fit_are_clipped(trans_b):
    sizes = [100, -5, 2 ** 31 - 1, 40]
    x, w, g, gs = _case([100, 0, 60, 0], 0, 64, 96, trans_b, torch.bfloat16)
    out = cc.grouped_matmul(x.cuda(), w.cuda(), torch.tensor(sizes, dtype=torch.int32).cuda(), trans_b=trans_b)
    grads = cc.grouped_matmul_backward(g.cuda(), x.cuda(), w.cuda(), torch.tensor(sizes, dtype=torch.int32).cuda(), trans_b=trans_b)
    _verify(out, x, w, sizes, trans_b, g, grads)


@pytest.mark.parametrize("experts", [64, 65, 200, 1024])
def test_many_groups(experts):
    gen = torch.Generator().manual_seed(experts)
    sizes = torch.randint(0, 4, (experts,), generator=gen).tolist()
    x, w, g, gs = _case(sizes, 5, 72, 48, 1, torch.bfloat16)
    grads = cc.grouped_matmul_backward(g.cuda(), x.cuda(), w.cuda(), gs.cuda(), trans_b=1)
    _verify(cc.grouped_matmul(x.cuda(), w.cuda(), gs.cuda(), trans_b=1), x, w, sizes, 1, g, grads)


@pytest.mark.parametrize("trans_b", [0, 1])
def test_what_belongs_to_others_does_not_reach_a_group(trans_b):
    """NaN and infinities in rows behind the last group, in experts without rows and in the other groups' rows leave a group's results as they are."""
    sizes, rest, k, n = [70, 0, 45, 130], 21, 136, 200
    x, w, g, gs = _case(sizes, rest, k, n, trans_b, torch.bfloat16)
    clean = [v.clone() for v in (x, w, g)]
    t = x.shape[0]
    x[t - rest:] = float("nan")
    g[t - rest:] = float("inf")
    w[1] = float("nan")
    x[70:115] = float("inf")
    g[70:115] = float("nan")
    out = cc.grouped_matmul(x.cuda(), w.cuda(), gs.cuda(), trans_b=trans_b)
    gx, gw = cc.grouped_matmul_backward(g.cuda(), x.cuda(), w.cuda(), gs.cuda(), trans_b=trans_b)
    want = cc.grouped_matmul(*(v.cuda() for v in clean[:2]), gs.cuda(), trans_b=trans_b)
    wx, ww = cc.grouped_matmul_backward(clean[2].cuda(), clean[0].cuda(), clean[1].cuda(), gs.cuda(), trans_b=trans_b)
    for rows in (slice(0, 70), slice(115, t)):
        assert torch.equal(out[rows], want[rows]) and torch.equal(gx[rows], wx[rows])
    for e in (0, 1, 3):
        assert torch.equal(gw[e], ww[e])
    assert not out[t - rest:].any() and not gx[t - rest:].any() and not gw[1].any()


def test_strided_and_unaligned_operands():
    x, w, g, gs = _case([50, 14], 0, 64, 48, 1, torch.bfloat16)
    want = cc.grouped_matmul(x.cuda(), w.cuda(), gs.cuda(), trans_b=1)
    wide = torch.zeros(64, 130, dtype=torch.bfloat16, device="cuda")
    wide[:, 1:129:2] = x.cuda()
    flat = torch.zeros(w.numel() + 1, dtype=torch.bfloat16, device="cuda")
    flat[1:] = w.cuda().flatten()
    assert torch.equal(cc.grouped_matmul(wide[:, 1:129:2], flat[1:].view(w.shape), gs.cuda(), trans_b=1), want)
    assert torch.equal(cc.grouped_matmul(x.cuda(), w.cuda().transpose(1, 2), gs.cuda(), trans_b=0), want)


@pytest.mark.parametrize("t,e,k,n", [(0, 3, 64, 32), (4, 2, 0, 16), (4, 2, 16, 0)])
def test_empty(t, e, k, n):
    x = torch.randn(t, k, device="cuda").bfloat16()
    w = torch.randn(e, k, n, device="cuda").bfloat16()
    gs = torch.tensor([t] + [0] * (e - 1), dtype=torch.int32, device="cuda")
    out = cc.grouped_matmul(x, w, gs)
    assert out.shape == (t, n) and not out.any()
    gx, gw = cc.grouped_matmul_backward(torch.ones(t, n, device="cuda").bfloat16(), x, w, gs)
    assert gx.shape == x.shape and gw.shape == w.shape and not gx.any() and not gw.any()


def test_one_gradient_alone():
    x, w, g, gs = (v.cuda() for v in _case([50, 14], 3, 64, 48, 1, torch.bfloat16))
    gx, gw = cc.grouped_matmul_backward(g, x, w, gs, trans_b=1)
    only = cc.grouped_matmul_backward(g, x, w, gs, trans_b=1, w_grad=False)
    assert only[1] is None and torch.equal(only[0], gx)
    only = cc.grouped_matmul_backward(g, x, w, gs, trans_b=1, x_grad=False)
    assert only[0] is None and torch.equal(only[1], gw)


def test_refusals():
    x, w, g, gs = (v.cuda() for v in _case([50, 14], 0, 64, 48, 1, torch.bfloat16))
    for bad in (lambda: cc.grouped_matmul(x.float(), w, gs, trans_b=1), lambda: cc.grouped_matmul(x, w.half(), gs, trans_b=1), lambda: cc.grouped_matmul(x, w, gs.long(), trans_b=1),
                lambda: cc.grouped_matmul(x, w, gs[:1], trans_b=1), lambda: cc.grouped_matmul(x, w, gs), lambda: cc.grouped_matmul(x, w[0], gs, trans_b=1),
                lambda: cc.grouped_matmul(x, w, gs, trans_b=2), lambda: cc.grouped_matmul(x.cpu(), w, gs, trans_b=1), lambda: cc.grouped_matmul(x, w, gs.cpu(), trans_b=1),
                lambda: cc.grouped_matmul_backward(g[:5], x, w, gs, trans_b=1), lambda: cc.grouped_matmul_backward(g.float(), x, w, gs, trans_b=1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(cc.CatccosError, match="num_experts"):
        cc.grouped_matmul(x, torch.zeros(1025, 48, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(1025, dtype=torch.int32, device="cuda"), trans_b=1)
