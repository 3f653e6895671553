"""torch.ops.catccos.* of the MoE gate, the balance loss and the 4-bit products under autograd, on Meta tensors: gradients where the Python entry points have them,
an error where they have none.  No GPU needed."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import catccos_amd.torch_library  # noqa: F401  (loads the library)

OPS = torch.ops.catccos


def meta(*shape, dtype=torch.float32, grad=False):
    return torch.empty(shape, dtype=dtype, device="meta", requires_grad=grad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("more", [False, True])
def test_gate_and_losses_have_gradients(dtype, more):
    logits = meta(30, 16, dtype=dtype, grad=True)
    bias, mask, offsets = (meta(16), meta(30, dtype=torch.bool), meta(4, dtype=torch.int32)) if more else (None, None, None)
    probs, idx = OPS.moe_router(logits, 4, "softmax", True, 1.0, bias, mask)
    assert probs.requires_grad and not idx.requires_grad
    loss, counts, tokens = OPS.moe_balance_loss(logits, idx, 0.1, 1e-3, "sigmoid", mask, offsets)
    assert loss.requires_grad and not counts.requires_grad and not tokens.requires_grad
    (loss + probs.sum()).backward()
    assert logits.grad.shape == logits.shape and logits.grad.dtype == dtype
    with torch.no_grad():
        assert not OPS.moe_router(logits, 4, "softmax", True, 1.0, bias, mask)[0].requires_grad
    assert not OPS.moe_router(logits.detach(), 4, "softmax", True, 1.0, bias, mask)[0].requires_grad


def test_second_derivatives_are_refused():
    logits = meta(30, 16, grad=True)
    for first in (lambda: OPS.moe_router(logits, 4, "softmax", True, 1.0, None, None)[0].sum(),
                  lambda: OPS.moe_balance_loss(logits, meta(30, 4, dtype=torch.int32), 0.1, 1e-3, "sigmoid", None, None)[0]):
        grad, = torch.autograd.grad(first(), logits, create_graph=True)
        with pytest.raises(RuntimeError, match="no gradient"):
            grad.sum().backward()


def test_products_have_none():
    u8 = lambda *shape: meta(*shape, dtype=torch.uint8)   # noqa: E731
    x, probs = meta(5, 256, dtype=torch.bfloat16, grad=True), meta(5, 2, grad=True)
    for of_x, of_probs in ((x, probs), (x.detach(), probs), (x, probs.detach())):
        out = OPS.moe_ffn_w4a16(of_x, meta(5, 2, dtype=torch.int32), of_probs, u8(4, 64, 128), u8(4, 64, 8), None, u8(4, 256, 16), u8(4, 256, 2), None, "e2m1", 32)
        assert out.requires_grad
        with pytest.raises(RuntimeError, match="no gradient"):
            out.sum().backward()
    out = OPS.w4a16_matmul(x, u8(96, 128), u8(96, 8), None, "e2m1", 32)
    with pytest.raises(RuntimeError, match="no gradient"):
        out.sum().backward()
    with torch.no_grad():
        assert not OPS.w4a16_matmul(x, u8(96, 128), u8(96, 8), None, "e2m1", 32).requires_grad
    assert not OPS.w4a16_matmul(x.detach(), u8(96, 128), u8(96, 8), None, "e2m1", 32).requires_grad


@pytest.mark.parametrize("recorded", [False, True])
def test_forward_mode_is_refused(recorded):
    u8 = lambda *shape: meta(*shape, dtype=torch.uint8)   # noqa: E731
    l, x = meta(30, 16, grad=recorded), meta(5, 256, dtype=torch.bfloat16, grad=recorded)
    with fwd.dual_level():
        d, dx = fwd.make_dual(l, torch.empty_like(l)), fwd.make_dual(x, torch.empty_like(x))
        for call in (lambda: OPS.moe_router(d, 4, "softmax", True, 1.0, None, None), lambda: OPS.moe_balance_loss(d, meta(30, 4, dtype=torch.int32), 0.1, 0.0, "softmax", None, None),
                     lambda: OPS.w4a16_matmul(dx, u8(96, 128), u8(96, 8), None, "e2m1", 32)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
