"""The 4-bit products have no derivatives: backward through them raises, and so does a call in forward mode; neither drops them."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import catccos_amd as cc
from catccos_amd import ops

pytestmark = pytest.mark.gpu


class Declines:
    def __getattr__(self, name):
        return lambda *a: NotImplemented


@pytest.fixture(params=["native", "general"])
def entry(request, monkeypatch):
    if request.param == "general":
        monkeypatch.setattr(ops, "_direct", Declines())


def products():
    gen = torch.Generator(device="cuda").manual_seed(1)

    def w(*shape):
        codes = torch.randint(0, 256, shape[:-1] + (shape[-1] // 2,), device="cuda", generator=gen, dtype=torch.uint8)
        return codes, (torch.rand(shape[:-1] + (shape[-1] // 32,), device="cuda", generator=gen) * 0.02).bfloat16(), None
    x = torch.randn(4, 64, device="cuda", generator=gen).bfloat16()
    probs, idx = cc.moe_router(torch.randn(4, 5, device="cuda", generator=gen), 2)
    dense, up, down = w(24, 64), w(5, 64, 64), w(5, 64, 32)
    return x, probs, lambda x, probs: cc.w4a16_matmul(x, *dense, group_size=32), lambda x, probs: cc.moe_ffn_w4a16(x, idx, probs, *up, *down, group_size=32)


@pytest.mark.parametrize("which,of_x,of_probs", [(0, True, False), (1, True, False), (1, False, True), (1, True, True)])
def test_the_products_have_no_gradient(entry, which, of_x, of_probs):
    x, probs, *calls = products()
    call = calls[which]
    want = call(x, probs)
    assert not want.requires_grad
    x, probs = x.clone().requires_grad_(of_x), probs.clone().requires_grad_(of_probs)
    out = call(x, probs)
    assert out.requires_grad and torch.equal(out, want)
    with pytest.raises(NotImplementedError, match="no gradient"):
        (out.float().sum() + x.float().sum() + probs.sum()).backward()
    for context in (torch.no_grad, torch.inference_mode):
        with context():
            quiet = call(x, probs)
        assert not quiet.requires_grad and torch.equal(quiet, want)
    with fwd.dual_level():
        tangent = (fwd.make_dual(x.detach(), torch.ones_like(x)) if of_x else x.detach(), fwd.make_dual(probs.detach(), torch.ones_like(probs)) if of_probs else probs.detach())
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(*tangent)
