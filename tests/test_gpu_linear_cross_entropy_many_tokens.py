"""linear_cross_entropy past 2^26 tokens, where a wave to a token would be more threads than a launch may have."""
import pytest
import torch

import catccos_amd as cc
from bounds16 import check, rounded, sum_error
from test_gpu_linear_cross_entropy import EXP

pytestmark = pytest.mark.gpu


def test_more_than_two_to_the_26_tokens():
    t, h, v = (1 << 26) + 5, 8, 24
    gen = torch.Generator(device="cuda").manual_seed(31)
    x = torch.empty(t, h, device="cuda", dtype=torch.bfloat16).normal_(generator=gen)
    w = torch.randn(v, h, device="cuda", generator=gen).bfloat16()
    tg = torch.randint(-4, v, (t,), device="cuda", generator=gen, dtype=torch.int32)
    loss, nll, lse, tokens = cc.linear_cross_entropy(x, w, tg)
    count = int((tg >= 0).sum())
    assert tokens.tolist() == [count]
    # a mean of float32 values in float64, rounded
    want = float(nll.sum(dtype=torch.float64)) / count
    assert abs(float(loss) - want) <= 2.0 ** -23 * abs(want)
    grad_x = cc.linear_cross_entropy_backward(torch.full((), float(count), device="cuda"), x, w, tg, lse, tokens, w_grad=False)[0]
    wd = w.double().cpu()
    for rows in (slice(0, 1000), slice((1 << 25) - 500, (1 << 25) + 500), slice(t - 1000, t)):
        xd, at = x[rows].double().cpu(), tg[rows].cpu().long()
        use = at >= 0
        l, el = xd @ wd.t(), sum_error(xd, wd.t())
        s = torch.logsumexp(l, 1)
        es = el.amax(1) + EXP + 128 * 2.0 ** -24 + 2.0 ** -22 * s.abs()
        pick = at.clamp_min(0)[:, None]
        n = s - l.gather(1, pick).squeeze(1)
        check(lse[rows], s * use, es * use, "lse")
        check(nll[rows], n * use, (es + el.gather(1, pick).squeeze(1) + 2.0 ** -23 * n.abs()) * use, "nll")
        # the mean's share times grad_loss is 1 up to float32's roundings of the number of tokens and of the quotient
        p = torch.exp(l - s[:, None])
        d = p.scatter_add(1, pick, torch.full_like(s, -1.0)[:, None]) * use[:, None]
        ed = (p * (2 * (el + es[:, None]) + EXP) + 2.0 ** -22 * d.abs()) * use[:, None]
        ed = ed + torch.finfo(torch.bfloat16).eps / 2 * (d.abs() + ed)
        y = d @ wd
        check(grad_x[rows], y, rounded(y, ed @ wd.abs() + sum_error(d.abs() + ed, wd) * 2 + 2.0 ** -21 * y.abs(), torch.bfloat16), "grad_x")
