"""matmul_bias_act and its gradients against float64, within bounds derived in bounds16.py and below."""
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

ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]
# The activations are smooth with a slope below 1.13 everywhere; computed in fp32 with a hardware exponential and reciprocal (a unit or two in the last place each, the exponent's
# argument off by 2^-22 of itself, and e^-z small where z is large) their own error stays below 2^-19 (|z| + 1).
SLOPE, OWN = 1.13, 2.0 ** -19


def _act(z, act):
    return {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
            "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[act](z)


def _case(m, k, n, trans_b, dtype, seed=1):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=gen).to(dtype)
    w = (torch.randn(*((n, k) if trans_b else (k, n)), generator=gen) * max(k, 1) ** -0.5).to(dtype)
    return x, w, torch.randn(n, generator=gen).to(dtype), torch.randn(m, n, generator=gen).to(dtype), torch.randn(m, n, generator=gen).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n,trans_b,act,bias,res", [
    (1, 64, 64, 1, "none", False, False), (1, 1024, 520, 1, "silu", True, True), (1, 1024, 520, 0, "gelu", True, True), (7, 72, 40, 1, "relu", True, False),
    (16, 256, 96, 0, "gelu_tanh", True, True), (17, 513, 65, 1, "silu", True, True), (33, 77, 131, 0, "gelu", False, True), (64, 2048, 136, 1, "gelu_tanh", True, False),
    (65, 8, 8, 1, "silu", True, True), (129, 320, 257, 1, "gelu", True, True), (300, 640, 384, 0, "gelu_tanh", True, True), (512, 192, 1000, 1, "none", True, False),
    (600, 1030, 770, 0, "silu", True, True), (1111, 130, 515, 1, "relu", False, True)])
def test_forward(m, k, n, trans_b, act, bias, res, dtype):
    x, w, b, r, _ = _case(m, k, n, trans_b, dtype)
    wk = (w.t() if trans_b else w).double()
    z = x.double() @ wk + (b.double() if bias else 0)
    ez = sum_error(x.double(), wk) + 2.0 ** -23 * z.abs()
    y = _act(z, act)
    ey = SLOPE * ez + (OWN * (z.abs() + 1) if act not in ("none", "relu") else 0)
    if res:
        y = y + r.double()
        ey = ey + 2.0 ** -23 * y.abs()
    args = (x.cuda(), w.cuda(), b.cuda() if bias else None, r.cuda() if res else None)
    out, pre = cc.matmul_bias_act(*args, activation=act, trans_b=trans_b, return_preact=True)
    check(out, y, rounded(y, ey, dtype), "out")
    check(pre, z, rounded(z, ez, dtype), "preact")
    assert torch.equal(cc.matmul_bias_act(*args, activation=act, trans_b=trans_b), out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n,trans_b,act", [(1, 64, 64, 1, "silu"), (7, 72, 40, 0, "relu"), (17, 513, 65, 1, "gelu"), (33, 77, 131, 0, "gelu_tanh"), (64, 512, 136, 1, "none"),
                                               (129, 320, 257, 1, "none"), (300, 640, 384, 0, "gelu_tanh"), (600, 264, 770, 1, "silu"), (1500, 96, 520, 0, "gelu")])
def test_backward(m, k, n, trans_b, act, dtype):
    x, w, _, pre, g = _case(m, k, n, trans_b, dtype)
    pre = pre * 2
    z = pre.double().requires_grad_()
    dz, = torch.autograd.grad(_act(z, act), z, g.double())
    # a slope's own error is below 2^-18 (it is below 1.13 and made of the same pieces), then dz is rounded
    ed = g.double().abs() * (2.0 ** -18 if act not in ("none", "relu") else 0)
    e16 = rounded(dz, ed, dtype) if act != "none" else torch.zeros_like(dz)
    wk, xd = (w.t() if trans_b else w).double(), x.double()
    gx = dz @ wk.t()
    bx = rounded(gx, e16 @ wk.abs().t() + sum_error(dz.abs() + e16, wk.t()), dtype)
    gw = xd.t() @ dz
    bw = rounded(gw, xd.abs().t() @ e16 + sum_error(xd.t(), dz.abs() + e16), dtype)
    if trans_b:
        gw, bw = gw.t(), bw.t()
    gb = dz.sum(0)
    bb = rounded(gb, (ed + m * 2.0 ** -23 * dz.abs()).sum(0), dtype)
    got = cc.matmul_bias_act_backward(g.cuda(), x.cuda(), w.cuda(), pre.cuda() if act != "none" else None, activation=act, trans_b=trans_b)
    for name, a, b, c in zip(("grad_x", "grad_w", "grad_bias"), got, (gx, gw, gb), (bx, bw, bb)):
        check(a, b, c, name)
    for only in range(3):
        want = [i == only for i in range(3)]
        part = cc.matmul_bias_act_backward(g.cuda(), x.cuda(), w.cuda(), pre.cuda(), activation=act, trans_b=trans_b, x_grad=want[0], w_grad=want[1], bias_grad=want[2])
        assert torch.equal(part[only], got[only]) and sum(v is not None for v in part) == 1


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("trans_b", [0, 1])
def test_autograd(act, trans_b):
    x, w, b, r, g = (v.cuda() for v in _case(130, 136, 72, trans_b, torch.bfloat16))
    leaves = [v.clone().requires_grad_() for v in (x, w, b, r)]
    out = cc.matmul_bias_act(*leaves, activation=act, trans_b=trans_b)
    out.backward(g)
    plain, pre = cc.matmul_bias_act(x, w, b, r, activation=act, trans_b=trans_b, return_preact=True)
    want = cc.matmul_bias_act_backward(g, x, w, pre, activation=act, trans_b=trans_b)
    assert torch.equal(out, plain)
    for leaf, v in zip(leaves, want + (g,)):
        assert torch.equal(leaf.grad, v)
    # some of them alone, and without a bias or a residual
    xr = x.clone().requires_grad_()
    cc.matmul_bias_act(xr, w, None, None, activation=act, trans_b=trans_b).backward(g)
    pre = cc.matmul_bias_act(x, w, activation=act, trans_b=trans_b, return_preact=True)[1]
    assert torch.equal(xr.grad, cc.matmul_bias_act_backward(g, x, w, pre, activation=act, trans_b=trans_b)[0])
    rr = r.clone().requires_grad_()
    cc.matmul_bias_act(x, w, None, rr, activation=act, trans_b=trans_b).backward(g)
    assert torch.equal(rr.grad, g)


@pytest.mark.parametrize("act", ACTS)
def test_against_differences(act):
    """The gradients of sum(out * g) in the direction d against differences of the float64 function whose values forward() is tested for: the analytic gradients here are
    those of that function up to the roundings of preact, dz and the results, each eps / 2 of its value (eps of preact changes the slope by at most 1.2 of |preact| eps / 2)."""
    x, w, b, r, g = _case(40, 48, 56, 1, torch.float16, seed=5)
    leaves = [v.cuda().requires_grad_() for v in (x, w, b, r)]
    cc.matmul_bias_act(*leaves, activation=act, trans_b=1).backward(g.cuda())
    gen = torch.Generator().manual_seed(9)

    def value(*v):
        return (_act(v[0] @ v[1].t() + v[2], act) + v[3]).mul(g.double()).sum()

    for i, leaf in enumerate(leaves):
        base = [v.double() for v in (x, w, b, r)]
        # an element near a kink of relu would spoil the difference: the direction touches a few elements, the step is small
        d = torch.zeros_like(base[i]).flatten()
        d[torch.randint(d.numel(), (8,), generator=gen)] = 1.0
        d = d.view(base[i].shape)
        h = 1e-6
        hi, lo = list(base), list(base)
        hi[i], lo[i] = base[i] + h * d, base[i] - h * d
        diff = (value(*hi) - value(*lo)) / (2 * h)
        z = base[0] @ base[1].t() + base[2]
        eps = torch.finfo(torch.float16).eps / 2
        terms = g.double().abs() * (SLOPE + 1.2 * z.abs()) * 3 * eps
        spread = {0: terms @ base[1].abs(), 1: terms.t() @ base[0].abs(), 2: terms.sum(0), 3: torch.zeros_like(base[3])}[i]
        got = (leaf.grad.double().cpu() * d).sum()
        assert abs(float(got - diff)) <= float((spread * d).sum()) + 2 * eps * float((leaf.grad.double().cpu().abs() * d).sum()) + 1e-5, (act, i)


@pytest.mark.parametrize("act", ACTS)
def test_values_far_out_and_not_finite(act):
    """A bias carries z far out: the activation and its slope have their limits, and a NaN stays in its column."""
    k, n = 16, 16
    z = torch.tensor([0.0, -0.0, 1e-3, 20.0, -20.0, 100.0, -100.0, 1e4, -1e4, 3e38, -3e38, float("nan"), 5.0, -5.0, 1.0, -1.0]).bfloat16()
    x, w = torch.zeros(4, k, dtype=torch.bfloat16), torch.zeros(n, k, dtype=torch.bfloat16)
    out = cc.matmul_bias_act(x.cuda(), w.cuda(), z.cuda(), activation=act, trans_b=1).cpu().double()
    zd = z.double()
    want = _act(zd, act)
    ok = ~torch.isnan(zd)
    assert (torch.isnan(out) == ~ok).all()
    assert ((out[:, ok] - want[ok]).abs() <= rounded(want[ok], OWN * (want[ok].abs() + 1), torch.bfloat16)).all()
    g = torch.ones(4, n, dtype=torch.bfloat16)
    pre = z.expand(4, n).contiguous()
    zr = zd.clone().requires_grad_()
    slope, = torch.autograd.grad(_act(zr, act)[ok].sum(), zr)
    gb = cc.matmul_bias_act_backward(g.cuda(), x.cuda(), w.cuda(), pre.cuda(), activation=act, trans_b=1)[2].cpu().double()
    slope = torch.where(zd.abs() > 1e30, (zd > 0).double() if act != "none" else torch.ones_like(zd), slope)
    assert ((gb[ok] - 4 * slope[ok]).abs() <= rounded(4 * slope[ok], torch.full_like(slope[ok], 4 * 2.0 ** -18), torch.bfloat16)).all()


@pytest.mark.parametrize("m,k,n", [(0, 16, 8), (4, 0, 8), (4, 16, 0)])
def test_empty(m, k, n):
    x, w, b, r, g = (v.cuda() for v in _case(m, k, n, 0, torch.bfloat16))
    out = cc.matmul_bias_act(x, w, b, r, activation="relu")
    assert out.shape == (m, n)
    if k == 0:
        want = (torch.relu(b.double()) + r.double()).cpu()
        check(out, want, rounded(want, 2.0 ** -23 * want.abs(), torch.bfloat16))
    gx, gw, gb = cc.matmul_bias_act_backward(g, x, w, r, activation="relu")
    assert gx.shape == x.shape and gw.shape == w.shape and gb.shape == b.shape
    if m == 0:
        assert not gw.any() and not gb.any()
    if n == 0:
        assert not gx.any()


def test_refusals():
    x, w, b, r, g = (v.cuda() for v in _case(20, 16, 24, 1, torch.bfloat16))
    for bad in (lambda: cc.matmul_bias_act(x, w), lambda: cc.matmul_bias_act(x.float(), w, trans_b=1), lambda: cc.matmul_bias_act(x, w.half(), trans_b=1),
                lambda: cc.matmul_bias_act(x, w, b[:3], trans_b=1), lambda: cc.matmul_bias_act(x, w, b.float(), trans_b=1), lambda: cc.matmul_bias_act(x, w, b, r[:3], trans_b=1),
                lambda: cc.matmul_bias_act(x, w, activation="tanh", trans_b=1), lambda: cc.matmul_bias_act(x, w.cpu(), trans_b=1),
                lambda: cc.matmul_bias_act_backward(g, x, w, None, activation="silu", trans_b=1), lambda: cc.matmul_bias_act_backward(g[:2], x, w, r, trans_b=1),
                lambda: cc.matmul_bias_act_backward(g, x, w, r[:2], activation="silu", trans_b=1)):
        with pytest.raises(ValueError):
            bad()
