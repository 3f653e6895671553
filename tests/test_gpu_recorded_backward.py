"""torch.ops.catccos: a backward pass that is recorded into a graph and would add to a leaf that an eager graph holds is refused by each operator's node.  Nothing is recorded here: the library
is told what to take the stream for."""
import pytest
import torch

import catccos_amd.torch_library  # noqa: F401

pytestmark = pytest.mark.gpu
OPS = torch.ops.catccos


@pytest.fixture
def library():
    assert OPS.init(0, 1, 1 << 20, "tcp://127.0.0.1:8666") == 0
    yield
    OPS._assume_recording(-1)
    assert OPS.finalize() == 0


def _case(op):
    """A leaf's values and what the operator makes of such a leaf."""
    gen = torch.Generator().manual_seed(1)
    x, w = torch.randn(8, 64, generator=gen).bfloat16().cuda(), torch.randn(2, 64, 32, generator=gen).bfloat16().cuda()
    sizes, tg = torch.tensor([5, 3], dtype=torch.int32).cuda(), torch.randint(2, (8,), generator=gen).cuda()
    return {"grouped_matmul": (w, lambda v: OPS.grouped_matmul(x, v, sizes, 0).sum()),
            "matmul_bias_act": (w[0].clone(), lambda v: OPS.matmul_bias_act(x, v, None, None, "silu", 0, False)[0].sum()),
            "matmul_bias_act, its residual": (w[0, :8].clone(), lambda v: OPS.matmul_bias_act(x, w[1], None, v, "none", 0, False)[0].sum()),
            "linear_cross_entropy": (x, lambda v: OPS.linear_cross_entropy(v, w[:, :, 0].contiguous(), tg, "mean", 0.0)[0])}[op]


@pytest.mark.parametrize("op", ["grouped_matmul", "matmul_bias_act", "matmul_bias_act, its residual", "linear_cross_entropy"])
def test_refused_where_a_leaf_is_held(library, op):
    value, of = _case(op)

    def grad(leaf, told):
        loss = of(leaf)
        OPS._assume_recording(told)
        try:
            loss.backward()
        finally:
            OPS._assume_recording(-1)
        return leaf.grad

    want = grad(value.clone().requires_grad_(), -1)
    with pytest.raises(RuntimeError, match="catccos::%s: .*eager graph" % op.split(",")[0]):
        grad(value.clone().requires_grad_(), 1)
    assert torch.equal(grad(value.clone().requires_grad_(), 0), want)
    # a leaf whose node was made on another stream, and one behind another node, are none of those
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [grad(value.clone().requires_grad_(), 1)]
        leaf = value.clone().requires_grad_()
        loss = of(leaf * 1)
        OPS._assume_recording(1)
        loss.backward()
        OPS._assume_recording(-1)
        got.append(leaf.grad)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, want) for g in got)


def test_what_it_is_told_is_answered_and_forgotten(library):
    assert OPS._assume_recording(1) == -1 and OPS._assume_recording(-1) == 1 and OPS._assume_recording(-1) == -1
