"""moe_balance_loss on both sides of the sizes where one workgroup is enough, with runs of several steps and with more runs than are added up at a time.
Formulas and tolerances: test_gpu_balance_loss."""
import pytest
import torch

from test_gpu_balance_loss import check, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,e,k", [(512, 16, 6), (513, 16, 6), (511, 30, 4), (256, 64, 8), (257, 64, 8), (256, 128, 8), (257, 128, 8), (128, 256, 8), (129, 256, 8),
                                   (64, 512, 8), (65, 500, 8), (32, 1024, 8), (33, 1024, 8)])
def test_one_workgroup_or_several(t, e, k, scoring):
    l, idx, gen = inputs(t + e, t, e, k, torch.float32)
    mask = (torch.rand(t, generator=gen) < 0.7).cuda()
    check(l, idx, 1.0, 0.01, scoring, mask=mask)
    _, _, tokens, grad = check(l, idx, 1.0, 0.01, scoring, offsets=[5, t - 3])
    assert int(tokens) == t - 8 and (grad[:5] == 0).all() and (grad[t - 3:] == 0).all()


@pytest.mark.parametrize("t,e,dtype", [(40000, 8, torch.bfloat16), (40000, 64, torch.float32), (20000, 200, torch.float16), (9000, 1000, torch.bfloat16)])
def test_many_tokens(t, e, dtype):
    l, idx, gen = inputs(t, t, e, 2, dtype)
    mask = (torch.rand(t, generator=gen) < 0.9).cuda()
    g = 2.0 ** 14 if dtype == torch.float16 else 1.0
    check(l, idx, 1.0, 0.001, "softmax", mask=mask, g=g)
    check(l, idx, 1.0, 0.0, "sigmoid", offsets=[0, t // 3, t // 3, t // 2 + 7, t], g=g)
