"""Forward-mode derivatives of the gate and the balance loss, which do not exist, are refused, not dropped."""
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


@pytest.mark.parametrize("recorded", [False, True])
def test_forward_mode_is_refused(entry, recorded):
    l = torch.randn(9, 16, device="cuda", requires_grad=recorded)
    _, idx = cc.moe_router(l.detach(), 3)
    with fwd.dual_level():
        d = fwd.make_dual(l, torch.ones_like(l))
        for call in (lambda: cc.moe_router(d, 3), lambda: cc.moe_router(d, 3, scoring="sigmoid", renormalize=False), lambda: cc.moe_balance_loss(d, idx),
                     lambda: cc.moe_balance_loss(d, idx, z_coef=0.1, scoring="sigmoid")):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        plain = cc.moe_router(l.detach(), 3)            # no tangent: as ever
        assert not plain[0].requires_grad and fwd.unpack_dual(plain[0]).tangent is None
    assert torch.equal(cc.moe_router(l.detach(), 3)[0], plain[0])
