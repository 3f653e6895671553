"""moe_router and its backward pass against the formulas in 64 bits.

Tolerances.  A weight is a quotient of exponentials: exp of an argument x in fp32 is off by up to |x| log2(e) 2^-23 relative (the product
with log2 e and that constant are rounded), for |x| <= 60 1.1e-5, sums and the division add 16 roundings of 2^-24: RTOL below.  A gradient is a difference of
products with the weights, so it is off by that times the largest |g| scale, and by half a unit of its type."""
import math

import pytest
import torch

import catccos_amd as cc

pytestmark = pytest.mark.gpu

RTOL = 60 * 1.4427 * 2.0 ** -23 + 16 * 2.0 ** -24
HALF_UNIT = {torch.float32: (0, 0), torch.bfloat16: (2.0 ** -8, 0), torch.float16: (2.0 ** -11, 2.0 ** -25)}


def reference(l, top_k, scoring, renorm, scale, bias=None, mask=None):
    """probs and experts of float64 logits, row by row."""
    l = l.double().cpu()
    probs, idx = torch.zeros(l.shape[0], top_k, dtype=torch.float64), torch.full((l.shape[0], top_k), -1, dtype=torch.int32)
    s = torch.sigmoid(l) if scoring == "sigmoid" else torch.softmax(l, 1)
    key = s + bias.double().cpu() if bias is not None else l
    for t in range(l.shape[0]):
        if mask is not None and not mask[t]:
            continue
        cand = [e for e in range(l.shape[1]) if l[t, e] > -math.inf]
        cand.sort(key=lambda e: (-float(key[t, e]), e))
        for j, e in enumerate(cand[:top_k]):
            idx[t, j] = e
            probs[t, j] = s[t, e]
    if renorm:
        if scoring == "softmax":   # the quotient, also where the scores themselves have left the range
            sel = torch.where(idx >= 0, l.gather(1, idx.clamp_min(0).long()), torch.tensor(-math.inf, dtype=torch.float64))
            probs = torch.softmax(sel, 1).nan_to_num(0.0)
        else:
            ls = torch.nn.functional.logsigmoid(l.gather(1, idx.clamp_min(0).long())).masked_fill(idx < 0, -math.inf)
            probs = torch.softmax(ls, 1).nan_to_num(0.0)
    return scale * probs, idx


def reference_grad(l, idx, g, scoring, renorm, scale):
    """Autograd in 64 bits through the selected scores."""
    l = l.double().cpu().requires_grad_()
    there = idx >= 0
    ls = torch.nn.functional.logsigmoid(l) if scoring == "sigmoid" else torch.log_softmax(l, 1)
    rows = there.any(1)
    sel = ls.gather(1, idx.clamp_min(0).long()).masked_fill(~there, -math.inf)[rows]
    w = torch.softmax(sel, 1) if renorm else torch.exp(sel)
    (scale * w * g.double().cpu()[rows]).sum().backward()
    return l.grad


def logits(seed, t, e, dtype):
    gen = torch.Generator().manual_seed(seed)
    return (2 * torch.randn(t, e, generator=gen)).to(dtype).cuda(), gen


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring,renorm,scale", [("softmax", True, 1.0), ("softmax", False, 1.0), ("sigmoid", True, 2.5), ("sigmoid", False, 0.5)])
@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (3, 2, 2), (65, 5, 3), (33, 16, 8), (40, 17, 6), (7, 60, 4), (129, 64, 8), (31, 100, 8), (20, 160, 6), (9, 256, 8),
                                   (5, 257, 2), (6, 512, 8), (3, 1000, 8), (2, 1024, 1)])
def test_weights_experts_and_gradient(t, e, k, scoring, renorm, scale, dtype):
    l, gen = logits(t + e, t, e, dtype)
    probs, idx = cc.moe_router(l, k, scoring=scoring, renormalize=renorm, scale=scale)
    assert probs.dtype == torch.float32 and idx.dtype == torch.int32
    want, want_idx = reference(l, k, scoring, renorm, scale)
    assert torch.equal(idx.cpu(), want_idx)
    assert ((probs.cpu().double() - want).abs() <= RTOL * want + 1e-30).all()
    g = torch.randn(t, k, generator=gen)
    got = cc.moe_router_backward(g.cuda(), l, idx, scoring=scoring, renormalize=renorm, scale=scale)
    assert got.dtype == dtype and got.shape == l.shape
    d = reference_grad(l, want_idx, g, scoring, renorm, scale)
    rel, abs_ = HALF_UNIT[dtype]
    assert ((got.cpu().double() - d).abs() <= rel * d.abs() + abs_ + 4 * RTOL * scale * float(g.abs().max())).all()


def test_ties_go_to_the_lower_index():
    l = torch.tensor([[1, 3, 3, 0, 3, 1, 1, 2.0] * 16, [0.0] * 128, [-0.0, 0.0] * 64])
    for dtype in (torch.float32, torch.bfloat16):
        _, idx = cc.moe_router(l.to(dtype).cuda(), 8)
        assert idx.cpu().tolist() == [[1, 2, 4, 9, 10, 12, 17, 18], list(range(8)), list(range(8))]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_masked_experts_masked_tokens_and_rows_without_any(scoring, renorm):
    l, gen = logits(3, 12, 24, torch.float32)
    l[1, 1:] = -math.inf          # one candidate
    l[2] = -math.inf              # none
    l[3, 4:] = -math.inf          # four for six routes
    l[4] = torch.finfo(torch.float32).min   # the type's lowest value is a value: all equal
    l[5] = torch.finfo(torch.float32).min
    l[5, 7] = 0.0
    l[:, 5] = -math.inf           # an expert that nobody gets
    l[6] = math.nan               # of a token that is masked: nothing of it may show
    l[7] = math.inf
    mask = torch.ones(12, dtype=torch.bool)
    mask[6] = mask[7] = mask[11] = False
    for m in (mask.cuda(), mask.to(torch.uint8).cuda()):
        probs, idx = cc.moe_router(l, 6, scoring=scoring, renormalize=renorm, token_mask=m)
    want, want_idx = reference(l, 6, scoring, renorm, 1.0, mask=mask)
    assert torch.equal(idx.cpu(), want_idx)
    assert (idx[2] == -1).all() and (idx[6] == -1).all() and idx[4].tolist() == [0, 1, 2, 3, 4, 6]
    assert ((probs.cpu().double() - want).abs() <= RTOL * want + 1e-30).all()
    g = torch.randn(12, 6, generator=gen)
    grad = cc.moe_router_backward(g.cuda(), l, idx, scoring=scoring, renormalize=renorm).cpu()
    assert (grad[[2, 6, 7, 11]] == 0).all() and (grad[:, 5] == 0).all() and torch.isfinite(grad).all()
    plain = [0, 1, 3, 8, 9, 10]
    d = reference_grad(l[plain], want_idx[plain], g[plain], scoring, renorm, 1.0)
    assert ((grad[plain].double() - d).abs() <= 4 * RTOL * float(g.abs().max())).all()


def test_nan_and_infinity_show_where_they_count_and_select_nothing_that_is_not_there():
    l = torch.zeros(2, 16, device="cuda")
    l[0, 3] = math.nan
    l[1, 3] = math.inf
    probs, idx = cc.moe_router(l, 4, renormalize=False)
    assert idx.tolist() == [[0, 1, 2, 4], [3, 0, 1, 2]]
    assert probs[0].isnan().all() and probs[1, 0].isnan()       # the softmax over all experts
    probs, idx = cc.moe_router(l, 4, scoring="sigmoid", renormalize=False)
    assert idx.tolist() == [[0, 1, 2, 4], [3, 0, 1, 2]] and probs.tolist() == [[0.5] * 4, [1.0, 0.5, 0.5, 0.5]]
    all_nan = torch.full((1, 16), math.nan, device="cuda")
    probs, idx = cc.moe_router(all_nan, 4)
    assert (idx == -1).all() and (probs == 0).all()


def test_logits_far_from_zero():
    for base in (-2000.0, -120.0, 120.0, 2000.0):
        l = base + torch.arange(32, device="cuda", dtype=torch.float32).flip(0).unsqueeze(0) / 8
        for scoring in ("softmax", "sigmoid"):
            probs, idx = cc.moe_router(l, 4, scoring=scoring)
            want, _ = reference(l, 4, scoring, True, 1.0)
            assert idx.tolist() == [[0, 1, 2, 3]]
            assert ((probs.cpu().double() - want).abs() <= RTOL * want).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e", [16, 72, 256])
def test_bias_selects_and_does_not_weigh(e, scoring):
    # scores and biases on grids on which no two sums are nearer than fp32 tells apart
    gen = torch.Generator().manual_seed(e)
    l = torch.randint(-12, 13, (50, e), generator=gen).float() / 4
    bias = torch.randint(-3, 4, (e,), generator=gen).float() * 0.0371
    s = torch.sigmoid(l.double()) if scoring == "sigmoid" else torch.softmax(l.double(), 1)
    key = s + bias.double()
    gaps = key.sort(1).values.diff(dim=1)
    usable = ((gaps > 1e-6) | (gaps < 1e-12)).all(1)
    assert usable.sum() > 20
    l, mask = l.cuda(), usable.cuda()
    probs, idx = cc.moe_router(l, 6, scoring=scoring, bias=bias.cuda(), token_mask=mask, scale=1.5)
    want, want_idx = reference(l, 6, scoring, True, 1.5, bias=bias, mask=usable)
    # equal sums in 64 bits may differ in the last bit there: compare what was chosen by key, and the lower index by equal logit and bias
    chosen = key.gather(1, idx.cpu().clamp_min(0).long())
    expect = key.gather(1, want_idx.clamp_min(0).long())
    assert ((chosen - expect).abs()[usable] <= 1e-6).all() and (idx.cpu()[~usable] == -1).all()
    got, _ = reference(l, 6, scoring, True, 1.5, bias=bias, mask=usable)
    same = (idx.cpu() == want_idx).all(1)
    assert ((probs.cpu().double() - got).abs()[same] <= RTOL * 1.5).all()
    hidden = bias.clone()
    hidden[2] = -math.inf
    _, idx = cc.moe_router(l, 6, scoring=scoring, bias=hidden.cuda())
    assert not (idx == 2).any()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_gradient_against_differences(scoring, renorm):
    # central differences of the kernel's own weights; logits 1/8 apart, so that a step of 1/64 changes no choice.  Truncation h^2/6 times a third
    # derivative of at most 1 per selected score, rounding 2 RTOL / (2 h)
    t, e, k, h = 6, 20, 4, 1.0 / 64
    gen = torch.Generator().manual_seed(1)
    l = torch.stack([torch.randperm(e, generator=gen) for _ in range(t)]).float().cuda() / 8
    g = torch.randn(t, k, generator=gen).cuda()
    _, idx = cc.moe_router(l, k, scoring=scoring, renormalize=renorm, scale=1.25)
    grad = cc.moe_router_backward(g, l, idx, scoring=scoring, renormalize=renorm, scale=1.25)
    for c in range(e):
        ends = []
        for sign in (1, -1):
            at = l.clone()
            at[:, c] += sign * h
            p, i = cc.moe_router(at, k, scoring=scoring, renormalize=renorm, scale=1.25)
            assert torch.equal(i, idx)
            ends.append((p.double() * g.double()).sum(1))
        diff = (ends[0] - ends[1]) / (2 * h)
        tol = 1.25 * k * float(g.abs().max()) * (h * h / 6 + RTOL / h)
        assert ((grad[:, c].double() - diff).abs() <= tol).all()


def test_autograd_strides_and_streams():
    base, gen = logits(9, 40, 64, torch.float32)
    l = base[::2, ::2].detach().requires_grad_()            # neither rows nor columns contiguous
    g = torch.randn(20, 4, generator=gen).cuda()
    probs, idx = cc.moe_router(l, 4, scale=2.0)
    assert probs.requires_grad and not idx.requires_grad
    (probs * g).sum().backward()
    flat = l.detach().contiguous()
    want, want_idx = cc.moe_router(flat, 4, scale=2.0)
    assert torch.equal(probs, want) and torch.equal(idx, want_idx)
    assert torch.equal(l.grad, cc.moe_router_backward(g, flat, idx, scale=2.0))
    with torch.no_grad():
        assert not cc.moe_router(l, 4)[0].requires_grad
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = cc.moe_router(flat, 4, scale=2.0)
    s.synchronize()
    assert torch.equal(other[0], want) and torch.equal(other[1], want_idx)


def test_rows_off_the_vector_boundaries():
    raw = torch.randn(33 * 64 + 1, device="cuda")
    l = raw[1:].view(33, 64)                                 # contiguous, 4 bytes past a 16-byte boundary
    for a, b in zip(cc.moe_router(l, 8), cc.moe_router(l.clone(), 8)):
        assert torch.equal(a, b)
    half = torch.randn(21 * 30 + 1, device="cuda").to(torch.bfloat16)[1:].view(21, 30)
    p, i = cc.moe_router(half, 3)
    q, j = cc.moe_router(half.clone(), 3)
    assert torch.equal(p, q) and torch.equal(i, j)
    g = torch.randn(21, 3, device="cuda")
    assert torch.equal(cc.moe_router_backward(g, half, i), cc.moe_router_backward(g, half.clone(), i))


def test_no_tokens():
    probs, idx = cc.moe_router(torch.empty(0, 16, device="cuda"), 2)
    assert probs.shape == idx.shape == (0, 2)
    assert cc.moe_router_backward(probs, torch.empty(0, 16, device="cuda"), idx).shape == (0, 16)


def test_routes_feed_the_sort():
    l, _ = logits(4, 50, 8, torch.float32)
    mask = torch.rand(50, device="cuda") < 0.7
    _, idx = cc.moe_router(l, 2, token_mask=mask)
    _, s2d, tokens = cc.moe_init_routing(idx, 8)
    assert int(tokens.sum()) == 2 * int(mask.sum()) and (s2d.view(50, 2)[~mask] == -1).all()


def test_refusals():
    l = torch.zeros(4, 16, device="cuda")
    for bad in (lambda: cc.moe_router(l.cpu(), 2), lambda: cc.moe_router(l.double(), 2), lambda: cc.moe_router(l[0], 2), lambda: cc.moe_router(l, 0),
                lambda: cc.moe_router(l, 9), lambda: cc.moe_router(l[:, :4], 5), lambda: cc.moe_router(l, 2, scoring="tanh"),
                lambda: cc.moe_router(l, 2, bias=torch.zeros(15, device="cuda")), lambda: cc.moe_router(l, 2, bias=torch.zeros(16, device="cuda").half()),
                lambda: cc.moe_router(l, 2, token_mask=torch.ones(3, dtype=torch.bool, device="cuda")),
                lambda: cc.moe_router(l, 2, token_mask=torch.ones(4, device="cuda")), lambda: cc.moe_router(l, 2, token_mask=torch.ones(4, dtype=torch.bool)),
                lambda: cc.moe_router_backward(torch.zeros(4, 2, device="cuda"), l, torch.zeros(4, 3, dtype=torch.int32, device="cuda")),
                lambda: cc.moe_router_backward(torch.zeros(4, 2, device="cuda"), l, torch.zeros(4, 2, dtype=torch.int64, device="cuda")),
                lambda: cc.moe_router_backward(torch.zeros(4, 2, device="cuda").half(), l, torch.zeros(4, 2, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(cc.CatccosError, match="num_experts"):
        cc.moe_router(torch.zeros(2, 1025, device="cuda"), 2)
