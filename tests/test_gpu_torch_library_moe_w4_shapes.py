"""torch.ops.catccos.* of the MoE gate and the 4-bit products: tensors with the right number of elements in another shape are refused, as in the Python entry points."""
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


def test_scales_in_another_order_are_refused(initialised):
    # [rows, experts, groups] has as many elements and groups as [experts, rows, groups]
    gen = torch.Generator(device="cuda").manual_seed(3)
    u8 = lambda *shape: torch.randint(0, 256, shape, device="cuda", generator=gen, dtype=torch.uint8)   # noqa: E731
    x = torch.randn(9, 256, device="cuda", generator=gen).bfloat16()
    w1, w2 = (u8(5, 128, 128), torch.rand(5, 128, 4, device="cuda").bfloat16()), (u8(5, 256, 32), torch.rand(5, 256, 1, device="cuda").bfloat16())
    probs, idx = cc.moe_router(torch.randn(9, 5, device="cuda", generator=gen), 3)
    ffn = lambda s1, s2: OPS.moe_ffn_w4a16(x, idx, probs, w1[0], s1, None, w2[0], s2, None, "int4", 64)   # noqa: E731
    ffn(w1[1], w2[1])
    for s1, s2 in ((w1[1].view(128, 5, 4), w2[1]), (w1[1], w2[1].view(256, 5, 1))):
        with pytest.raises(RuntimeError, match="scales of"):
            ffn(s1, s2)
    router = lambda b, m: OPS.moe_router(probs, 2, "softmax", True, 1.0, b, m)   # noqa: E731
    for b, m in ((torch.zeros(3, 1, device="cuda"), None), (None, torch.ones(3, 3, dtype=torch.bool, device="cuda"))):
        with pytest.raises(RuntimeError):
            router(b, m)
    with pytest.raises(ValueError):
        cc.moe_router(probs, 2, bias=torch.zeros(3, 1, device="cuda"))
