"""Calls that are more than one launch because a grid's dimension ends: results on both sides of each split, and the whole of them.  Tolerances: test_gpu_w4a16, test_gpu_router."""
import pytest
import torch

import catccos_amd as cc
from test_gpu_router import RTOL
from test_gpu_w4a16 import check_block, check_product, weights

pytestmark = pytest.mark.gpu


def rows_of_x(seed, m, k):
    return torch.randn(m, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).bfloat16()


@pytest.mark.parametrize("fmt,group,zeros", [("int4", 32, True), ("e2m1", 32, False)])
def test_dense_rows_past_the_grid(fmt, group, zeros):
    # 16 rows to a tile, 65535 tiles to a launch
    m, k, n = 65535 * 16 + 5, 32, 2
    check_product(rows_of_x(1, m, k), weights(torch.Generator().manual_seed(1), (n,), k, fmt, group, zeros, torch.bfloat16), fmt, group)


@pytest.mark.parametrize("fmt,group,zeros", [("int4", 32, True), ("e2m1", 32, False)])
def test_rows_of_any_k_past_the_grid(fmt, group, zeros):
    m, k, n = 65540, 33, 3
    check_product(rows_of_x(2, m, k), weights(torch.Generator().manual_seed(2), (n,), k, fmt, group, zeros, torch.bfloat16), fmt, group)


@pytest.mark.parametrize("k,n,top_k", [(32, 64, 1), (33, 6, 1), (32, 64, 3)])
def test_tokens_of_the_block_past_the_grid(k, n, top_k):
    m, e = 65540, 3
    gen = torch.Generator().manual_seed(k)
    w1, w2 = weights(gen, (e, n), k, "int4", 32, True, torch.bfloat16), weights(gen, (e, k), n // 2, "int4", 32, True, torch.bfloat16)
    idx = torch.stack([torch.randperm(e, generator=gen)[:top_k] for _ in range(97)]).repeat(m // 97 + 1, 1)[:m].int().cuda()
    probs = torch.rand(m, top_k, generator=gen).cuda()
    check_block(rows_of_x(3, m, k), idx, probs, w1, w2, "int4", 32)


def test_router_tokens_past_one_launch():
    t, e = (1 << 25) + 5, 3
    gen = torch.Generator(device="cuda").manual_seed(4)
    l = torch.randint(-40, 41, (t, e), device="cuda", generator=gen).bfloat16() / 8
    mask = torch.rand(t, device="cuda", generator=gen) < 0.9
    probs, idx = cc.moe_router(l, 1, scoring="sigmoid", renormalize=False, scale=2.0, token_mask=mask)
    best = torch.where(l[:, 0] >= torch.maximum(l[:, 1], l[:, 2]), 0, torch.where(l[:, 1] >= l[:, 2], 1, 2))     # (ties to the lower index)
    assert torch.equal(idx[:, 0], torch.where(mask, best, -1).int())
    s = torch.sigmoid(l.float().amax(1).double())
    assert ((probs[:, 0].double() - 2 * s).abs()[mask] <= RTOL * 2 * s[mask]).all() and (probs[~mask] == 0).all()
    g = torch.randn(t, 1, device="cuda", generator=gen)
    grad = cc.moe_router_backward(g, l, idx, scoring="sigmoid", renormalize=False, scale=2.0)
    own = torch.where(mask, 2 * s * (1 - s) * g[:, 0].double(), 0.0)
    d = torch.zeros(t, e, dtype=torch.float64, device="cuda").scatter_(1, best.unsqueeze(1), own.unsqueeze(1))
    assert ((grad.double() - d).abs() <= 2.0 ** -8 * d.abs() + 8 * RTOL * float(g.abs().max())).all()
