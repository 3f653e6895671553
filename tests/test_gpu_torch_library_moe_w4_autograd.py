"""torch.ops.catccos.* of the MoE gate and the balance loss under autograd on the GPU: the gradients of the Python entry points, to the bit."""
import pytest
import torch

import catccos_amd as cc
import catccos_amd.torch_library  # noqa: F401

pytestmark = pytest.mark.gpu
OPS = torch.ops.catccos


@pytest.fixture
def initialised():
    assert OPS.finalize() == 0
    assert OPS.init(0, 1, 1 << 20, "tcp://127.0.0.1:8666") == 0
    yield
    assert OPS.finalize() == 0


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gradients(initialised, dtype, scoring):
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = torch.randn(77, 40, device="cuda", generator=g).to(dtype)
    bias, mask = torch.randn(40, device="cuda", generator=g) * 0.1, torch.rand(77, device="cuda", generator=g) < 0.9
    offsets, grad = torch.tensor([0, 20, 20, 70], dtype=torch.int32, device="cuda"), torch.randn(77, 4, device="cuda", generator=g)
    for b, m, off in ((None, None, None), (bias, mask, offsets)):
        got = []
        for lib in (OPS, cc):
            leaf = logits.clone().requires_grad_()
            probs, idx = lib.moe_router(leaf, 4, scoring, False, 2.0, b, m)
            (probs * grad).sum().backward()
            got.append([probs.detach(), idx, leaf.grad])
            leaf = logits.clone().requires_grad_()
            loss, counts, tokens = lib.moe_balance_loss(leaf, idx, 0.1, 1e-3, scoring, m, off)
            (3 * loss).backward()
            got[-1] += [loss.detach(), counts, tokens, leaf.grad]
        assert all(torch.equal(a, w) for a, w in zip(*got)) and got[0][2].abs().sum() > 0 and got[0][6].abs().sum() > 0
