"""torch.ops.catccos.* of the products of 16-bit operands, the dense layer and the loss: Meta shapes, gradients on Meta tensors, refusals.  No GPU needed."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import catccos_amd.torch_library  # noqa: F401  (loads the library)

OPS = torch.ops.catccos
BF = torch.bfloat16


def meta(*shape, dtype=BF, grad=False):
    return torch.empty(shape, dtype=dtype, device="meta", requires_grad=grad)


def i32(*shape):
    return meta(*shape, dtype=torch.int32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_shapes(dtype):
    x, g = meta(30, 64, dtype=dtype), meta(30, 48, dtype=dtype)
    like = lambda t, *shape: t.dtype == dtype and tuple(t.shape) == shape   # noqa: E731
    for trans_b in (0, 1):
        w3, w2 = (meta(*s, dtype=dtype) for s in (((4, 48, 64), (48, 64)) if trans_b else ((4, 64, 48), (64, 48))))
        assert like(OPS.grouped_matmul(x, w3, i32(4), trans_b), 30, 48)
        gx, gw = OPS.grouped_matmul_backward(g, x, w3, i32(4), trans_b, True, False)
        assert like(gx, 30, 64) and like(gw, 0)
        gx, gw = OPS.grouped_matmul_backward(g, x, w3, i32(4), trans_b, False, True)
        assert like(gx, 0) and like(gw, *w3.shape)
        out, pre = OPS.matmul_bias_act(x, w2, meta(48, dtype=dtype), g, "gelu", trans_b, True)
        assert like(out, 30, 48) and like(pre, 30, 48) and like(OPS.matmul_bias_act(x, w2, None, None, "none", trans_b, False)[1], 0)
        gx, gw, gb = OPS.matmul_bias_act_backward(g, x, w2, pre, "gelu", trans_b, True, True, True)
        assert like(gx, 30, 64) and like(gw, *w2.shape) and like(gb, 48)
    w, tg = meta(1000, 64, dtype=dtype), meta(30, dtype=torch.int64)
    loss, nll, lse, tokens = OPS.linear_cross_entropy(x, w, tg, "mean", 0.0)
    assert loss.shape == () and nll.shape == lse.shape == (30,) and tokens.shape == (1,) and loss.dtype == nll.dtype == lse.dtype == torch.float32 and tokens.dtype == torch.int32
    gx, gw = OPS.linear_cross_entropy_backward(loss, x, w, tg, lse, tokens, "sum", 0.0, True, True)
    assert like(gx, 30, 64) and like(gw, 1000, 64)


def test_gradients_where_they_are_wanted():
    x, w = meta(30, 64, grad=True), meta(4, 64, 48, grad=True)
    OPS.grouped_matmul(x, w, i32(4), 0).sum().backward()
    assert x.grad.shape == x.shape and w.grad.shape == w.shape
    x = meta(30, 64, grad=True)
    OPS.grouped_matmul(x, w.detach(), i32(4), 0).sum().backward()
    assert x.grad.shape == x.shape
    for act in ("none", "silu"):
        leaves = [meta(30, 64, grad=True), meta(48, 64, grad=True), meta(48, grad=True), meta(30, 48, grad=True)]
        for some in range(1, 16):
            ins = [v if some >> i & 1 else v.detach() for i, v in enumerate(leaves)]
            out, pre = OPS.matmul_bias_act(*ins, act, 1, bool(some & 1))
            assert out.requires_grad and not pre.requires_grad and pre.shape == ((30, 48) if some & 1 else (0,))
            out.sum().backward()
            for i, v in enumerate(leaves):
                assert (v.grad is not None) == bool(some >> i & 1) and (v.grad is None or v.grad.shape == v.shape)
                v.grad = None
    x, w = meta(30, 64, grad=True), meta(1000, 64, grad=True)
    loss, nll, lse, tokens = OPS.linear_cross_entropy(x, w, meta(30, dtype=torch.int64), "mean", 1e-3)
    assert loss.requires_grad and not (nll.requires_grad or lse.requires_grad or tokens.requires_grad)
    loss.backward()
    assert x.grad.shape == x.shape and w.grad.shape == w.shape
    with torch.no_grad():
        assert not OPS.linear_cross_entropy(x, w, meta(30, dtype=torch.int64), "mean", 1e-3)[0].requires_grad


def test_second_derivatives_are_refused():
    x, w3, w2 = meta(30, 64, grad=True), meta(4, 64, 48), meta(64, 48)
    for first in (lambda: OPS.grouped_matmul(x, w3, i32(4), 0).sum(), lambda: OPS.matmul_bias_act(x, w2, None, None, "gelu", 0, False)[0].sum(),
                  lambda: OPS.linear_cross_entropy(x, meta(100, 64), meta(30, dtype=torch.int64), "mean", 0.0)[0]):
        grad, = torch.autograd.grad(first(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="no gradient"):
            grad.sum().backward()


@pytest.mark.parametrize("recorded", [False, True])
def test_forward_mode_is_refused(recorded):
    x, w3, w2, tg = meta(30, 64, grad=recorded), meta(4, 64, 48), meta(64, 48), meta(30, dtype=torch.int64)
    with fwd.dual_level():
        d = fwd.make_dual(x, meta(30, 64))
        for call in (lambda: OPS.grouped_matmul(d, w3, i32(4), 0), lambda: OPS.matmul_bias_act(d, w2, None, None, "none", 0, False),
                     lambda: OPS.linear_cross_entropy(d, meta(100, 64), tg, "mean", 0.0)):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()


def test_host_tensors_find_no_kernel():
    x, w = torch.zeros(4, 16, dtype=BF), torch.zeros(2, 16, 8, dtype=BF)
    for call in (lambda: OPS.grouped_matmul(x, w, torch.zeros(2, dtype=torch.int32), 0), lambda: OPS.matmul_bias_act(x, w[0], None, None, "none", 0, False),
                 lambda: OPS.linear_cross_entropy(x, x, torch.zeros(4, dtype=torch.int64), "mean", 0.0)):
        with pytest.raises(NotImplementedError):
            call()
    with pytest.raises(RuntimeError, match="activation"):
        OPS.matmul_bias_act(meta(4, 16), meta(16, 8), None, None, "tanh", 0, False)
    with pytest.raises(RuntimeError, match="reduction"):
        OPS.linear_cross_entropy(meta(4, 16), meta(8, 16), meta(4, dtype=torch.int64), "none", 0.0)
