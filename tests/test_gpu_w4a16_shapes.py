"""w4a16_matmul and moe_ffn_w4a16 at the row and column counts where the kernels change their workgroups, with zero points past the codes' own range and with K so long
that the scales do not fit LDS at once.  Formulas and tolerances: test_gpu_w4a16."""
import pytest
import torch

import catccos_amd as cc
from test_gpu_w4a16 import KINDS, activations, block, check_block, check_product, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,group,zeros", KINDS)
@pytest.mark.parametrize("m,n", [(1, 8192), (4, 8208), (5, 8192), (8, 8193), (9, 4096), (16, 4112), (16, 8200), (13, 16400), (16, 32784), (17, 8192), (32, 8224), (31, 16420),
                                 (33, 4128), (64, 8220), (65, 10960), (96, 16000)])
def test_columns(m, n, fmt, group, zeros):
    gen = torch.Generator().manual_seed(m + n)
    check_product(activations(gen, m, 288, torch.bfloat16), weights(gen, (n,), 288, fmt, group, zeros, torch.bfloat16), fmt, group)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(1, 48, 40960), (7, 40, 40960), (16, 24, 40960), (20, 33, 24576), (70, 64, 24576), (70, 16400, 4224)])
def test_scales_in_several_pieces(m, n, k, dtype):
    gen = torch.Generator().manual_seed(m + n)
    check_product(activations(gen, m, k, dtype), weights(gen, (n,), k, "int4", 32, True, dtype), "int4", 32)


@pytest.mark.parametrize("dtype,highest", [(torch.bfloat16, 240), (torch.float16, 255)])
@pytest.mark.parametrize("m,k", [(1, 256), (16, 256), (40, 256), (3, 100)])
def test_zero_points_past_the_codes(m, k, dtype, highest):
    gen = torch.Generator().manual_seed(m)
    w, s, _ = weights(gen, (48,), k, "int4", 64, False, dtype)
    z = torch.randint(0, highest + 1, s.shape, generator=gen, dtype=torch.uint8).cuda()
    z[0], z[1] = highest, 16
    check_product(activations(gen, m, k, dtype), (w, s, z), "int4", 64)


@pytest.mark.parametrize("fmt,group,zeros", KINDS)
@pytest.mark.parametrize("m,e,top_k", [(4, 6, 3), (5, 6, 3), (16, 2, 2), (17, 40, 4), (32, 3, 2), (40, 6, 2), (80, 4, 2)])
def test_routes_of_an_expert(m, e, top_k, fmt, group, zeros):
    check_block(*block(m + e, m, 224, 384, e, top_k, fmt, group, zeros, torch.bfloat16), fmt, group)


@pytest.mark.parametrize("top_k", range(1, 9))
@pytest.mark.parametrize("k", [64, 66])
def test_every_number_of_routes_is_combined(top_k, k):
    x, idx, probs, w1, w2 = block(top_k, 9, k, 32, 10, top_k, "int4", 32, False, torch.float16)
    idx[2, 0] = -1
    check_block(x, idx, probs, w1, w2, "int4", 32)
