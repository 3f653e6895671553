"""Scale bytes that belong to no element: the second of a pair behind K's last group (MXFP4 rows of an odd number of groups), and groups of other parts of K.

An MXFP4 row has 2 * ceil(K / 64) scale bytes, so where K is an odd multiple of 32 the last is padding.  Whatever it holds, results are the same bits."""
import math

import pytest
import torch

import catccos_amd as cc
from test_gpu_w4a16 import activations, block, check_block, check_product, weights

pytestmark = pytest.mark.gpu


def padded(w, byte):
    codes, s, z = w
    s = s.clone()
    s[..., -1] = byte
    return codes, s, z


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k", [32, 96, 160, 544, 2016, 7200])
@pytest.mark.parametrize("m,n", [(1, 40), (1, 9000), (7, 48), (16, 80), (30, 64), (64, 100), (130, 4200)])
def test_product(m, n, k, dtype):
    gen = torch.Generator().manual_seed(m * n + k)
    x, w = activations(gen, m, k, dtype), weights(gen, (n,), k, "e2m1", 32, False, dtype)
    want = check_product(x, padded(w, 127), "e2m1", 32)
    for byte in (255, 254, 0):
        assert torch.equal(cc.w4a16_matmul(x, *padded(w, byte), fmt="e2m1"), want), byte


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n,e,top_k", [(1, 96, 64, 3, 2), (2, 160, 320, 8, 4), (20, 544, 192, 6, 3), (40, 96, 64, 2, 1), (60, 160, 192, 4, 2), (100, 224, 64, 2, 2)])
def test_block(m, k, n, e, top_k, dtype):
    x, idx, probs, w1, w2 = block(m + k, m, k, n, e, top_k, "e2m1", 32, False, dtype)
    want = check_block(x, idx, probs, padded(w1, 127), padded(w2, 127), "e2m1", 32)     # (k and n / 2 are odd multiples of 32)
    for one, two in ((255, 127), (127, 255), (255, 254)):
        assert torch.equal(cc.moe_ffn_w4a16(x, idx, probs, *padded(w1, one), *padded(w2, two), fmt="e2m1"), want)


def test_any_k_does_not_read_it_either():
    gen = torch.Generator().manual_seed(1)
    for k in (1, 31, 65, 90, 129):                       # one, three or five groups
        x, w = activations(gen, 3, k, torch.bfloat16), weights(gen, (20,), k, "e2m1", 32, False, torch.bfloat16)
        assert torch.equal(cc.w4a16_matmul(x, *padded(w, 255), fmt="e2m1"), cc.w4a16_matmul(x, *padded(w, 127), fmt="e2m1"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 8, 16, 20, 64])
def test_an_infinite_scale_stays_an_infinity(m, group, zeros, dtype):
    # nine blocks of 128 in two, four or eight parts: some parts have a block less, and none may meet a neighbour's scale.  x > 0 and the largest codes: the sum is +inf
    k, n = 9 * 128, 33
    gen = torch.Generator().manual_seed(m)
    x = activations(gen, m, k, dtype).abs() + 0.5
    codes = torch.full((n, k // 2), 0xFF, dtype=torch.uint8, device="cuda")
    s = torch.full((n, k // group), 0.01, dtype=dtype, device="cuda")
    z = torch.full((n, k // group), 3, dtype=torch.uint8, device="cuda") if zeros else None
    clean = cc.w4a16_matmul(x, codes, s, z, group_size=group)
    for at in range(k // group):
        some = s.clone()
        some[at % n, at] = math.inf
        out = cc.w4a16_matmul(x, codes, some, z, group_size=group)
        assert (out[:, at % n] == math.inf).all(), at
        rest = [i for i in range(n) if i != at % n]
        assert torch.equal(out[:, rest], clean[:, rest])
