"""moe_balance_loss and its backward pass against the formulas in 64 bits.

Tolerances.  A share p is a quotient of exponentials whose arguments stay below 60: off by RTOL relative (the product with log2 e and that constant
are rounded, then sums and divisions), and so are their means and sums, all of one sign, with a rounding of 2^-24 per addition: a workgroup's wave adds at most
tokens / 4 values one after the other.  lse is off by RTOL absolute and its rounding.  A gradient is p times a difference of routes' shares: RTOL of p times
the largest share, and half a unit of its type."""
import math

import pytest
import torch

import catccos_amd as cc

pytestmark = pytest.mark.gpu

RTOL = 60 * 1.4427 * 2.0 ** -23 + 16 * 2.0 ** -24
HALF_UNIT = {torch.float32: (0, 0), torch.bfloat16: (2.0 ** -8, 0), torch.float16: (2.0 ** -11, 2.0 ** -25)}


def reference(l, idx, coef, z_coef, scoring, mask=None, offsets=None):
    """loss (with autograd), counts, tokens and the largest unit of a token's gradient, of float64 logits."""
    t, e = l.shape
    use = torch.ones(t, dtype=torch.bool) if mask is None else mask.cpu().bool()
    use = use & (l.detach() > -math.inf).any(1)
    cuts = [0, t] if offsets is None else offsets
    spans = list(zip(cuts[:-1], cuts[1:]))
    counts, tokens, parts, z = torch.zeros(len(spans), e, dtype=torch.int32), torch.zeros(len(spans), dtype=torch.int32), [], []
    unit = 0.0
    for s, (a, b) in enumerate(spans):
        rows = [i for i in range(a, b) if use[i]]
        tokens[s] = len(rows)
        if not rows:
            continue
        i = idx[rows].flatten().long()
        counts[s] = torch.bincount(i[(i >= 0) & (i < e)], minlength=e).int()
        x = l[rows]
        p = torch.softmax(x if scoring == "softmax" else torch.nn.functional.logsigmoid(x), 1)
        f = counts[s].double() * e / (idx.shape[1] * len(rows))
        parts.append((f * p.mean(0)).sum())
        z.append((torch.logsumexp(x, 1) ** 2).sum())
        unit = max(unit, float(f.max()) / len(rows))
    n = max(1, int(tokens.sum()))
    loss = (coef * sum(parts) / len(parts) + z_coef * sum(z) / n) if parts else torch.zeros((), dtype=torch.float64)
    return loss, counts, tokens, coef * unit / max(1, len(parts)), z_coef * 2 / n


def check(l, idx, coef, z_coef, scoring, mask=None, offsets=None, g=1.0):
    dev = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device="cuda")
    opt = {"coef": coef, "z_coef": z_coef, "scoring": scoring, "token_mask": mask, "seq_offsets": dev}
    loss, counts, tokens = cc.moe_balance_loss(l, idx, **opt)
    ref = l.double().cpu().requires_grad_()
    want, wc, wt, unit, zunit = reference(ref, idx.cpu(), coef, z_coef, scoring, mask, offsets)
    assert loss.shape == () and loss.dtype == torch.float32 and counts.dtype == tokens.dtype == torch.int32
    assert torch.equal(counts.cpu(), wc if offsets is not None else wc[0]) and torch.equal(tokens.cpu(), wt)
    adds = (l.shape[0] / 4 + 300) * 2.0 ** -24
    assert abs(float(loss) - float(want)) <= (2 * RTOL + adds) * float(want) + 1e-30
    again = cc.moe_balance_loss(l, idx, **opt)
    assert all(torch.equal(a, b) for a, b in zip((loss, counts, tokens), again))
    grad = cc.moe_balance_loss_backward(torch.tensor(g, device="cuda"), l, counts, tokens, idx.shape[1], **opt)
    assert grad.dtype == l.dtype and grad.shape == l.shape
    if want.requires_grad:
        want.backward()
    d = g * ref.grad.nan_to_num(0.0) if ref.grad is not None else torch.zeros_like(ref)
    biggest = float(torch.logsumexp(ref.detach(), 1).abs().nan_to_num(0.0, posinf=0.0, neginf=0.0).max()) if l.numel() else 0.0
    rel, abs_ = HALF_UNIT[l.dtype]
    tol = rel * d.abs() + abs_ + 8 * RTOL * g * (unit + zunit * (biggest + 1))
    assert ((grad.cpu().double() - d).abs() <= tol).all()
    return loss, counts, tokens, grad


def inputs(seed, t, e, k, dtype):
    gen = torch.Generator().manual_seed(seed)
    l = (2 * torch.randn(t, e, generator=gen) + torch.randn(e, generator=gen)).to(dtype)
    return l.cuda(), l.float().topk(k, dim=1).indices.int().cuda(), gen


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("z_coef", [0.0, 0.01])
@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 16, 4), (2, 2, 2), (67, 5, 3), (300, 16, 6), (33, 33, 2), (1025, 64, 8), (50, 100, 8), (77, 256, 8), (31, 257, 4),
                                   (9, 640, 8), (5, 1024, 8)])
def test_loss_counts_and_gradient(t, e, k, z_coef, scoring, dtype):
    l, idx, _ = inputs(t * e, t, e, k, dtype)
    check(l, idx, 0.5, z_coef, scoring, g=2.0 ** 12 if dtype == torch.float16 else 1.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,e,offsets", [(100, 16, [0, 100]), (100, 16, [0, 0, 1, 2, 50, 50, 99, 100, 100]), (100, 72, [7, 30, 64, 90]), (700, 256, [0, 1, 600, 700]),
                                         (40, 8, [40, 40]), (3, 32, [0, 1, 2, 3])])
def test_sequences_of_all_lengths_and_tokens_in_none(t, e, offsets, scoring):
    l, idx, gen = inputs(t + e, t, e, 3, torch.float32)
    mask = (torch.rand(t, generator=gen) < 0.8).cuda()
    for m in (None, mask):
        _, _, _, grad = check(l, idx, 1.0, 0.001, scoring, mask=m, offsets=offsets)
        assert (grad[:offsets[0]] == 0).all() and (grad[offsets[-1]:] == 0).all()


def test_many_sequences():
    l, idx, _ = inputs(5, 1500, 20, 2, torch.float32)
    check(l, idx, 1.0, 0.0, "softmax", offsets=list(range(0, 1501, 3)))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_rows_with_nothing_masked_rows_and_dropped_routes(scoring):
    l, idx, _ = inputs(6, 40, 24, 4, torch.float32)
    l[3] = -math.inf                       # no expert there: does not count
    l[4, 1:] = -math.inf
    l[5, ::2] = -math.inf
    l[6] = torch.finfo(torch.float32).min  # the lowest value is a value: equal shares
    l[7] = math.nan
    l[8] = math.inf
    idx[9] = -1
    idx[10, 1] = 24
    idx[11, 2] = 1 << 30
    mask = torch.ones(40, dtype=torch.bool, device="cuda")
    mask[7] = mask[8] = False              # whatever a masked row holds
    _, counts, tokens, grad = check(l, idx, 1.0, 0.0, scoring, mask=mask)
    assert int(tokens) == 37 and int(counts.sum()) == 36 * 4 - 2
    assert (grad[[3, 7, 8]] == 0).all() and torch.isfinite(grad).all()
    none = torch.zeros(40, dtype=torch.bool, device="cuda")
    loss, counts, tokens, grad = check(l, idx, 1.0, 0.5, scoring, mask=none)
    assert float(loss) == 0 and int(tokens) == 0 and (counts == 0).all() and (grad == 0).all()


def test_nan_in_a_counted_row_shows():
    l, idx, _ = inputs(6, 40, 24, 4, torch.float32)
    l[3, 2] = math.nan
    loss, counts, tokens = cc.moe_balance_loss(l, idx)
    assert loss.isnan() and int(tokens) == 40 and int(counts.sum()) == 160


def test_logits_far_from_zero():
    for base in (-2000.0, -110.0, 110.0, 2000.0):
        l, idx, _ = inputs(8, 30, 32, 2, torch.float32)
        l = (l * 8).round() / 8 + base
        for scoring in ("softmax", "sigmoid"):
            check(l, idx, 1.0, 0.0, scoring)


def test_balanced_routing_has_loss_one():
    # equal logits: P = 1/E for every expert, f = 1 on average
    e = 16
    idx = torch.arange(64, dtype=torch.int32, device="cuda").view(32, 2) % e
    loss, counts, _ = cc.moe_balance_loss(torch.zeros(32, e, device="cuda"), idx)
    assert abs(float(loss) - 1) < 1e-6 and (counts == 4).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_gradient_against_differences(scoring):
    # central differences of the formula's own loss in 64 bits: truncation h^2/6 times a third derivative of at most 6 units, rounding 1e-15 / h
    l, idx, gen = inputs(11, 12, 10, 3, torch.float32)
    _, counts, tokens, grad = check(l, idx, 1.0, 0.05, scoring, offsets=[0, 5, 12])
    h = 1e-4
    for _ in range(40):
        t, e = int(torch.randint(12, (1,), generator=gen)), int(torch.randint(10, (1,), generator=gen))
        ends = []
        for sign in (1, -1):
            x = l.double().cpu()
            x[t, e] += sign * h
            loss, _, _, unit, zunit = reference(x, idx.cpu(), 1.0, 0.05, scoring, None, [0, 5, 12])
            ends.append(float(loss))
        tol = 8 * RTOL * (unit + 20 * zunit) + h * h * (unit + 20 * zunit) + 1e-10
        assert abs(float(grad[t, e]) - (ends[0] - ends[1]) / (2 * h)) <= tol


def test_autograd_strides_and_streams():
    base, _, _ = inputs(9, 64, 48, 2, torch.float32)
    l = base[::2, ::2].detach().requires_grad_()
    idx = torch.randint(0, 24, (32, 4), dtype=torch.int32, device="cuda")[:, ::2]
    off = torch.tensor([0, 9, 32], dtype=torch.int32, device="cuda")
    loss, counts, tokens = cc.moe_balance_loss(l, idx, coef=0.3, z_coef=0.2, seq_offsets=off)
    assert loss.requires_grad and not counts.requires_grad and not tokens.requires_grad
    (3 * loss).backward()
    flat = l.detach().contiguous()
    want = cc.moe_balance_loss(flat, idx.contiguous(), coef=0.3, z_coef=0.2, seq_offsets=off)
    assert all(torch.equal(a, b) for a, b in zip((loss, counts, tokens), want))
    assert torch.equal(l.grad, cc.moe_balance_loss_backward(torch.tensor(3.0, device="cuda"), flat, counts, tokens, 2, coef=0.3, z_coef=0.2, seq_offsets=off))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = cc.moe_balance_loss(flat, idx.contiguous(), coef=0.3, z_coef=0.2, seq_offsets=off)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))


def test_no_tokens():
    l, idx = torch.empty(0, 16, device="cuda"), torch.empty(0, 2, dtype=torch.int32, device="cuda")
    loss, counts, tokens = cc.moe_balance_loss(l, idx, z_coef=1.0)
    assert float(loss) == 0 and (counts == 0).all() and int(tokens) == 0
    assert cc.moe_balance_loss_backward(torch.ones((), device="cuda"), l, counts, tokens, 2).shape == (0, 16)


def test_rows_off_the_vector_boundaries():
    raw = torch.randn(33 * 64 + 1, device="cuda")
    l = raw[1:].view(33, 64)
    idx = torch.randint(0, 64, (33, 2), dtype=torch.int32, device="cuda")
    a, b = cc.moe_balance_loss(l, idx), cc.moe_balance_loss(l.clone(), idx)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    g = torch.ones((), device="cuda")
    assert torch.equal(cc.moe_balance_loss_backward(g, l, *a[1:], 2), cc.moe_balance_loss_backward(g, l.clone(), *a[1:], 2))


def test_refusals():
    l, idx = torch.zeros(4, 16, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    one = torch.ones((), device="cuda")
    for bad in (lambda: cc.moe_balance_loss(l.cpu(), idx), lambda: cc.moe_balance_loss(l, idx.cpu()), lambda: cc.moe_balance_loss(l.double(), idx),
                lambda: cc.moe_balance_loss(l, idx.long()), lambda: cc.moe_balance_loss(l, idx[:3]), lambda: cc.moe_balance_loss(l, idx[0]),
                lambda: cc.moe_balance_loss(l, idx, scoring="relu"), lambda: cc.moe_balance_loss(l, idx, token_mask=torch.ones(5, dtype=torch.bool, device="cuda")),
                lambda: cc.moe_balance_loss(l, idx, seq_offsets=i32(0)), lambda: cc.moe_balance_loss(l, idx, seq_offsets=i32(0, 4).long()),
                lambda: cc.moe_balance_loss_backward(one.double(), l, i32(*[0] * 16), i32(4), 2), lambda: cc.moe_balance_loss_backward(one, l, i32(*[0] * 15), i32(4), 2),
                lambda: cc.moe_balance_loss_backward(one, l, i32(*[0] * 16), i32(4, 4), 2),
                lambda: cc.moe_balance_loss_backward(one, l, i32(*[0] * 16), i32(4), 2, seq_offsets=i32(0, 2, 4))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(cc.CatccosError, match="num_experts"):
        cc.moe_balance_loss(torch.zeros(4, 1025, device="cuda"), idx)
    with pytest.raises(cc.CatccosError, match="top_k"):
        cc.moe_balance_loss_backward(one, l, i32(*[0] * 16), i32(4), 9)
