"""torch.ops.catccos.* of the MoE gate, the balance loss and the 4-bit products on the GPU: the bits of the Python entry points, and their refusals."""
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


def same(a, b):
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8))


def gate(dtype):
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = torch.randn(77, 40, device="cuda", generator=g).to(dtype)
    return (logits, torch.randn(40, device="cuda", generator=g) * 0.1, torch.rand(77, device="cuda", generator=g) < 0.9,
            torch.tensor([0, 20, 20, 70], dtype=torch.int32, device="cuda"), torch.randn(77, 4, device="cuda", generator=g))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gate_and_losses(initialised, dtype, scoring):
    logits, bias, mask, offsets, grad = gate(dtype)
    one = torch.tensor(0.5, device="cuda")
    for b, m in ((None, None), (bias, mask)):
        probs, idx = OPS.moe_router(logits, 4, scoring, True, 2.0, b, m)
        for got, want in zip((probs, idx), cc.moe_router(logits, 4, scoring, True, 2.0, b, m)):
            assert same(got, want)
        assert same(OPS.moe_router_backward(grad, logits, idx, scoring, True, 2.0), cc.moe_router_backward(grad, logits, idx, scoring, True, 2.0))
        for off in (None, offsets):
            got = OPS.moe_balance_loss(logits, idx, 0.1, 1e-3, scoring, m, off)
            for a, w in zip(got, cc.moe_balance_loss(logits, idx, 0.1, 1e-3, scoring, m, off)):
                assert same(a, w)
            assert same(OPS.moe_balance_loss_backward(one, logits, *got[1:], 4, 0.1, 1e-3, scoring, m, off),
                        cc.moe_balance_loss_backward(one, logits, *got[1:], 4, 0.1, 1e-3, scoring, m, off))
    wide = torch.stack([logits, logits], 2)[..., 0]                        # strides are made contiguous
    assert same(OPS.moe_router(wide, 4, scoring, True, 2.0, None, None)[0], cc.moe_router(logits, 4, scoring, True, 2.0)[0])


def weights(gen, lead, k, fmt, group, zeros, dtype):
    codes = torch.randint(0, 256, lead + (k // 2,), device="cuda", generator=gen, dtype=torch.uint8)
    if fmt == "e2m1":
        return codes, torch.randint(118, 124, lead + (cc.scale_cols(k),), device="cuda", generator=gen, dtype=torch.uint8), None
    s = (torch.rand(lead + ((k + group - 1) // group,), device="cuda", generator=gen) * 0.02).to(dtype)
    return codes, s, torch.randint(0, 16, s.shape, device="cuda", generator=gen, dtype=torch.uint8) if zeros else None


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt,group,zeros", [("int4", 128, True), ("int4", 32, False), ("e2m1", 32, False)])
def test_products(initialised, fmt, group, zeros, dtype):
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(9, 256, device="cuda", generator=gen).to(dtype)
    w = weights(gen, (72,), 256, fmt, group, zeros, dtype)
    assert same(OPS.w4a16_matmul(x, *w, fmt, group), cc.w4a16_matmul(x, *w, fmt=fmt, group_size=group))
    w1, w2 = weights(gen, (5, 128), 256, fmt, group, zeros, dtype), weights(gen, (5, 256), 64, fmt, group, zeros, dtype)
    probs, idx = OPS.moe_router(torch.randn(9, 5, device="cuda", generator=gen), 3, "softmax", True, 1.0, None, None)
    assert same(OPS.moe_ffn_w4a16(x, idx, probs, *w1, *w2, fmt, group), cc.moe_ffn_w4a16(x, idx, probs, *w1, *w2, fmt=fmt, group_size=group))


def test_refusals(initialised):
    logits, bias, mask, offsets, grad = gate(torch.float32)
    probs, idx = OPS.moe_router(logits, 4, "softmax", True, 1.0, None, None)
    loss, counts, tokens = OPS.moe_balance_loss(logits, idx, 1.0, 0.0, "softmax", None, None)
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(2, 256, device="cuda", generator=gen).bfloat16()
    w, s, z = weights(gen, (8,), 256, "int4", 64, True, torch.bfloat16)
    router = lambda *a: OPS.moe_router(*a)   # noqa: E731
    for bad in (lambda: router(logits, 9, "softmax", True, 1.0, None, None), lambda: router(logits, 4, "none", True, 1.0, None, None),
                lambda: router(logits.double(), 4, "softmax", True, 1.0, None, None), lambda: router(logits, 4, "softmax", True, 1.0, bias.cpu(), None),
                lambda: router(logits, 4, "softmax", True, 1.0, bias[:3], None), lambda: router(logits, 4, "softmax", True, 1.0, None, mask.float()),
                lambda: OPS.moe_router_backward(grad.cpu(), logits, idx, "softmax", True, 1.0), lambda: OPS.moe_router_backward(grad[:, :3], logits, idx, "softmax", True, 1.0),
                lambda: OPS.moe_balance_loss(logits, idx.long(), 1.0, 0.0, "softmax", None, None), lambda: OPS.moe_balance_loss(logits, idx, 1.0, 0.0, "softmax", None, offsets.long()),
                lambda: OPS.moe_balance_loss(logits, idx.cpu(), 1.0, 0.0, "softmax", None, None),
                lambda: OPS.moe_balance_loss_backward(loss, logits, counts[:3], tokens, 4, 1.0, 0.0, "softmax", None, None),
                lambda: OPS.w4a16_matmul(x, w.cpu(), s, z, "int4", 64), lambda: OPS.w4a16_matmul(x, w, s, z.cpu(), "int4", 64), lambda: OPS.w4a16_matmul(x, w, s, z, "int8", 64),
                lambda: OPS.w4a16_matmul(x, w, s, z, "int4", 48), lambda: OPS.w4a16_matmul(x, w[:, :5], s, z, "int4", 64), lambda: OPS.w4a16_matmul(x, w, s.half(), z, "int4", 64),
                lambda: OPS.w4a16_matmul(x, w, s, z[:4], "int4", 64), lambda: OPS.w4a16_matmul(x.float(), w, s, z, "int4", 64)):
        with pytest.raises(RuntimeError):
            bad()
    assert OPS.finalize() == 0
    with pytest.raises(RuntimeError, match="not initialized"):
        router(logits, 4, "softmax", True, 1.0, None, None)
