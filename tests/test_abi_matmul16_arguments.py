"""Argument checks of the products of 16-bit operands and of the loss that return before any device work: they run without a GPU."""
import pytest

from catccos_amd import _abi

P = 0x1000   # a non-null pointer that is never dereferenced: every call below fails its checks first, or has nothing to do
BIG = 1 << 40   # a workspace that is large enough for anything below


def rejected(rc, *needles):
    msg = _abi.lib().cch_last_error().decode()
    assert rc == _abi.EINVAL, (rc, msg)
    for n in needles:
        assert n in msg, msg


def grouped(x=P, w=P, sizes=P, out=P, e=4, t=64, n=32, k=16, trans_b=0, dtype=0, ws=P, nbytes=BIG):
    return _abi.lib().cch_grouped_matmul(x, w, sizes, out, e, t, n, k, trans_b, dtype, ws, nbytes, None)


def grouped_backward(grad=P, x=P, w=P, sizes=P, grad_x=P, grad_w=P, e=4, t=64, n=32, k=16, trans_b=0, dtype=0, ws=P, nbytes=BIG):
    return _abi.lib().cch_grouped_matmul_backward(grad, x, w, sizes, grad_x, grad_w, e, t, n, k, trans_b, dtype, ws, nbytes, None)


def layer(x=P, w=P, bias=None, residual=None, preact=None, out=P, t=64, n=32, k=16, trans_b=0, act=0, dtype=0, ws=P, nbytes=BIG):
    return _abi.lib().cch_matmul_bias_act(x, w, bias, residual, preact, out, t, n, k, trans_b, act, dtype, ws, nbytes, None)


def layer_backward(grad=P, x=P, w=P, preact=None, grad_x=P, grad_w=P, grad_bias=P, t=64, n=32, k=16, trans_b=0, act=0, dtype=0, ws=P, nbytes=BIG):
    return _abi.lib().cch_matmul_bias_act_backward(grad, x, w, preact, grad_x, grad_w, grad_bias, t, n, k, trans_b, act, dtype, ws, nbytes, None)


def loss(x=P, w=P, targets=P, target_bytes=8, out=P, nll=P, lse=P, tokens=P, t=64, h=16, v=100, reduction=0, dtype=0, ws=P, nbytes=BIG):
    return _abi.lib().cch_linear_cross_entropy(x, w, targets, target_bytes, out, nll, lse, tokens, t, h, v, reduction, 0.0, dtype, ws, nbytes, None)


def loss_backward(grad=P, x=P, w=P, targets=P, target_bytes=8, lse=P, tokens=P, grad_x=P, grad_w=P, t=64, h=16, v=100, reduction=0, dtype=0, ws=P, nbytes=BIG):
    return _abi.lib().cch_linear_cross_entropy_backward(grad, x, w, targets, target_bytes, lse, tokens, grad_x, grad_w, t, h, v, reduction, 0.0, dtype, ws, nbytes, None)


@pytest.mark.parametrize("call,name", [(grouped, "cch_grouped_matmul:"), (grouped_backward, "cch_grouped_matmul_backward:"), (layer, "cch_matmul_bias_act:"),
                                       (layer_backward, "cch_matmul_bias_act_backward:")])
def test_products(call, name):
    for bad in ({"t": -1}, {"n": -1}, {"k": -1}, {"t": (1 << 30) + 1}, {"n": (1 << 22) + 1}, {"k": (1 << 22) + 1}):
        rejected(call(**bad), name, "shape")
    rejected(call(trans_b=2), name, "trans_b=2")
    rejected(call(dtype=2), name, "type 2")
    rejected(call(dtype=-1), name, "type -1")
    rejected(call(x=None), name, "null")
    rejected(call(w=None), name, "null")
    rejected(call(x=P + 2), name, "16-byte")
    rejected(call(w=P + 8), name, "16-byte")
    rejected(call(k=17, n=33, ws=None), name, "workspace")
    rejected(call(k=17, n=33, ws=P + 128), name, "workspace")
    rejected(call(k=17, n=33, nbytes=1), name, "workspace")


@pytest.mark.parametrize("call", [grouped, grouped_backward])
def test_groups(call):
    rejected(call(e=0), "num_experts=0")
    rejected(call(e=1025), "num_experts=1025")
    rejected(call(sizes=None), "null")
    assert grouped(t=0, x=None, out=None) == _abi.OK and grouped(n=0, w=None, out=None) == _abi.OK
    assert grouped_backward(grad_x=None, grad_w=None, k=16, n=32) == _abi.OK


@pytest.mark.parametrize("call", [layer, layer_backward])
def test_activations(call):
    rejected(call(act=-1), "activation -1")
    rejected(call(act=5), "activation 5")
    rejected(layer_backward(act=2), "null")
    rejected(layer(out=None), "null")
    rejected(layer_backward(grad=None), "null")
    rejected(layer(bias=P + 1), "odd")
    rejected(layer(residual=P + 1), "odd")
    rejected(layer(preact=P + 1), "odd")
    rejected(layer_backward(grad_bias=P + 1), "odd")
    assert layer(t=0, x=None, out=None) == _abi.OK and layer(n=0, w=None, out=None) == _abi.OK


@pytest.mark.parametrize("call,name", [(loss, "cch_linear_cross_entropy:"), (loss_backward, "cch_linear_cross_entropy_backward:")])
def test_loss(call, name):
    for bad in ({"t": -1}, {"t": (1 << 30) + 1}, {"h": 0}, {"h": (1 << 22) + 1}, {"v": 0}, {"v": (1 << 30) + 1}):
        rejected(call(**bad), name, "shape")
    rejected(call(target_bytes=2), name, "2 bytes")
    rejected(call(reduction=2), name, "reduction 2")
    rejected(call(dtype=2), name, "type 2")
    for null in ("x", "w", "targets", "lse", "tokens"):
        rejected(call(**{null: None}), name, "null")
    rejected(loss(out=None), "null")
    rejected(loss(nll=None), "null")
    rejected(loss_backward(grad=None), "null")
    rejected(call(x=P + 8), name, "16-byte")
    rejected(call(w=P + 8), name, "16-byte")
    rejected(call(targets=P + 4), name)
    rejected(call(ws=None), name, "workspace")
    rejected(call(ws=P + 128), name, "workspace")
    rejected(call(nbytes=255), name, "workspace")
    assert loss_backward(grad_x=None, grad_w=None) == _abi.OK


def test_workspaces_of_what_is_refused_are_empty():
    L = _abi.lib()
    assert L.cch_grouped_matmul_workspace_bytes(0, 64, 33, 17, 0) == 0 == L.cch_grouped_matmul_backward_workspace_bytes(1025, 64, 33, 17, 0)
    assert L.cch_matmul_bias_act_workspace_bytes(-1, 33, 17, 0) == 0 == L.cch_matmul_bias_act_backward_workspace_bytes(1 << 31, 33, 17, 0, 2)
    assert L.cch_linear_cross_entropy_workspace_bytes(4, 0, 8) == 0 == L.cch_linear_cross_entropy_backward_workspace_bytes(4, 8, 0)
    # the largest shapes: no overflow
    assert L.cch_grouped_matmul_backward_workspace_bytes(1024, 1 << 30, (1 << 22) - 1, (1 << 22) - 1, 1) > 1 << 50
    assert L.cch_linear_cross_entropy_backward_workspace_bytes(1 << 30, (1 << 22) - 1, 1 << 30) > 1 << 50


def test_the_kernel_option():
    L = _abi.lib()
    for value in (-1, 0, 1, 2):
        assert L.cch_set_option(b"matmul16_kernel", value) == _abi.OK
    rejected(L.cch_set_option(b"matmul16_kernel", 3))
    rejected(L.cch_set_option(b"matmul16_kernel", -2))
    assert L.cch_set_option(b"matmul16_kernel", -1) == _abi.OK
