"""torch.ops.catccos.* of the MoE gate, the balance loss and the 4-bit products: registration, init state, Meta shapes.  No GPU needed."""
import pytest
import torch

import catccos_amd.torch_library  # noqa: F401  (loads the library)

OPS = torch.ops.catccos


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("name", ["moe_router", "moe_router_backward", "moe_balance_loss", "moe_balance_loss_backward", "w4a16_matmul", "moe_ffn_w4a16"])
def test_registration(name):
    assert hasattr(OPS, name)
    for key, there in (("CUDA", True), ("Meta", True), ("CPU", False)):
        assert torch._C._dispatch_has_kernel_for_dispatch_key("catccos::" + name, key) == there


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_meta_shapes_of_gate_and_losses(dtype):
    logits, mask, offsets = meta(300, 64, dtype=dtype), meta(300, dtype=torch.bool), meta(5, dtype=torch.int32)
    probs, idx = OPS.moe_router(logits, 8, "sigmoid", True, 2.5, meta(64, dtype=torch.float32), mask)
    assert probs.shape == idx.shape == (300, 8) and probs.dtype == torch.float32 and idx.dtype == torch.int32 and probs.device.type == "meta"
    grad = OPS.moe_router_backward(probs, logits, idx, "sigmoid", True, 2.5)
    assert grad.shape == logits.shape and grad.dtype == dtype
    for off, shape, s in ((None, (64,), 1), (offsets, (4, 64), 4)):
        loss, counts, tokens = OPS.moe_balance_loss(logits, idx, 0.1, 0.0, "softmax", mask, off)
        assert loss.shape == () and loss.dtype == torch.float32 and counts.shape == shape and counts.dtype == torch.int32 and tokens.shape == (s,)
        grad = OPS.moe_balance_loss_backward(loss, logits, counts, tokens, 8, 0.1, 0.0, "softmax", mask, off)
        assert grad.shape == logits.shape and grad.dtype == dtype


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_meta_shapes_of_products(dtype):
    u8 = lambda *shape: meta(*shape, dtype=torch.uint8)   # noqa: E731
    x = meta(5, 256, dtype=dtype)
    out = OPS.w4a16_matmul(x, u8(96, 128), meta(96, 2, dtype=dtype), u8(96, 2), "int4", 128)
    assert out.shape == (5, 96) and out.dtype == dtype and out.device.type == "meta"
    assert OPS.w4a16_matmul(x, u8(96, 128), u8(96, 8), None, "e2m1", 32).shape == (5, 96)
    out = OPS.moe_ffn_w4a16(x, meta(5, 2, dtype=torch.int32), meta(5, 2, dtype=torch.float32), u8(4, 64, 128), u8(4, 64, 8), None, u8(4, 256, 16), u8(4, 256, 2), None, "e2m1", 32)
    assert out.shape == (5, 256) and out.dtype == dtype


def test_cpu_tensors_have_no_kernel():
    with pytest.raises(NotImplementedError):
        OPS.moe_router(torch.zeros(4, 8), 2, "softmax", True, 1.0, None, None)
    with pytest.raises(NotImplementedError):
        OPS.w4a16_matmul(torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 1, dtype=torch.bfloat16), None, "int4", 64)
