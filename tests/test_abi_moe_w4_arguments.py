"""Argument checks of the router, the balance loss and the 4-bit products that return before any device work: they run without a GPU."""
from catccos_amd import _abi

P = 0x1000   # a non-null pointer that is never dereferenced: every call below fails its checks first
BIG = 1 << 31


def rejected(rc, *needles):
    msg = _abi.lib().cch_last_error().decode()
    assert rc == _abi.EINVAL, (rc, msg)
    for n in needles:
        assert n in msg, msg


def router(logits=P, dtype=0, tokens=4, experts=8, top_k=2, scoring=0, renormalize=1, probs=P, idx=P):
    return _abi.lib().cch_moe_router(logits, dtype, tokens, experts, top_k, scoring, renormalize, 1.0, None, None, probs, idx, None)


def router_backward(grad=P, logits=P, dtype=0, idx=P, tokens=4, experts=8, top_k=2, scoring=0, renormalize=1, out=P):
    return _abi.lib().cch_moe_router_backward(grad, logits, dtype, idx, tokens, experts, top_k, scoring, renormalize, 1.0, out, None)


def test_router_arguments():
    for call, name in ((router, "cch_moe_router:"), (router_backward, "cch_moe_router_backward:")):
        rejected(call(dtype=3), name, "type 3")
        rejected(call(tokens=-1), name, "tokens")
        rejected(call(tokens=(1 << 30) + 1), name, "tokens")
        rejected(call(experts=0), name, "num_experts")
        rejected(call(experts=1025), name, "num_experts")
        rejected(call(top_k=0), name, "top_k")
        rejected(call(top_k=9, experts=16), name, "top_k")
        rejected(call(top_k=4, experts=3), name, "top_k")
        rejected(call(scoring=2), name, "scoring")
        rejected(call(renormalize=2), name, "renormalize")
        rejected(call(logits=None), name, "null")
        rejected(call(idx=None), name, "null")
        assert call(tokens=0, logits=None, idx=None) == _abi.OK
    rejected(router(probs=None), "null")
    rejected(router_backward(grad=None), "null")
    rejected(router_backward(out=None), "null")


def balance(logits=P, dtype=0, idx=P, offsets=None, tokens=4, experts=8, top_k=2, sequences=1, scoring=0, loss=P, counts=P, seq_tokens=P, workspace=P, nbytes=None):
    L = _abi.lib()
    if nbytes is None:
        nbytes = L.cch_moe_balance_loss_workspace_bytes(tokens, experts, sequences)
    return L.cch_moe_balance_loss(logits, dtype, idx, None, offsets, tokens, experts, top_k, sequences, scoring, 1.0, 0.0, loss, counts, seq_tokens, workspace, nbytes, None)


def balance_backward(grad=P, logits=P, dtype=0, offsets=None, counts=P, seq_tokens=P, tokens=4, experts=8, top_k=2, sequences=1, scoring=0, out=P):
    return _abi.lib().cch_moe_balance_loss_backward(grad, logits, dtype, None, offsets, counts, seq_tokens, tokens, experts, top_k, sequences, scoring, 1.0, 0.0, out, None)


def test_balance_loss_arguments():
    L = _abi.lib()
    for call, name in ((balance, "cch_moe_balance_loss:"), (balance_backward, "cch_moe_balance_loss_backward:")):
        rejected(call(dtype=-1), name, "type -1")
        rejected(call(tokens=-1), name, "tokens")
        rejected(call(tokens=(1 << 30) + 1, top_k=1), name, "tokens")
        rejected(call(tokens=1 << 29, top_k=4), name, "routes")
        rejected(call(experts=0), name, "num_experts")
        rejected(call(experts=1025), name, "num_experts")
        rejected(call(top_k=9), name, "top_k")
        rejected(call(sequences=0, offsets=P), name, "num_sequences")
        rejected(call(sequences=2), name, "num_sequences")                 # no offsets
        rejected(call(sequences=65536, offsets=P), name, "num_sequences")
        rejected(call(scoring=-1), name, "scoring")
        rejected(call(logits=None), name, "null")
        rejected(call(counts=None), name, "null")
        rejected(call(seq_tokens=None), name, "null")
    rejected(balance(idx=None), "null")
    rejected(balance(loss=None), "null")
    rejected(balance(workspace=None), "workspace")
    rejected(balance(nbytes=8), "workspace of 8 bytes")
    rejected(balance(workspace=P + 2), "workspace")
    rejected(balance_backward(grad=None), "null")
    assert balance_backward(tokens=0, logits=None) == _abi.OK
    assert L.cch_moe_balance_loss_workspace_bytes(-1, 8, 1) == 0 and L.cch_moe_balance_loss_workspace_bytes(4, 2000, 1) == 0
    assert 0 < L.cch_moe_balance_loss_workspace_bytes(0, 8, 1) <= L.cch_moe_balance_loss_workspace_bytes(1 << 20, 8, 1)


INT4, E2M1 = _abi.FMT_INT4, _abi.FMT_E2M1


def product(x=P, w=P, s=P, z=None, out=P, m=4, n=8, k=64, fmt=INT4, group=32, dtype=0):
    return _abi.lib().cch_w4a16_matmul(x, w, s, z, out, m, n, k, fmt, group, dtype, None, 0, None)


def test_w4a16_matmul_arguments():
    rejected(product(m=-1), "cch_w4a16_matmul", "shape")
    rejected(product(m=BIG), "shape")
    rejected(product(n=(1 << 25) + 1), "shape")
    rejected(product(k=1 << 30), "shape")
    rejected(product(fmt=0), "format 0")
    rejected(product(group=48), "group_size 48")
    rejected(product(dtype=2), "type 2")                                   # activations are 16-bit
    for missing in ("x", "w", "s", "out"):
        rejected(product(**{missing: None}), "null")
    assert product(m=0, x=None, out=None) == _abi.OK and product(n=0, w=None) == _abi.OK
    assert _abi.lib().cch_w4a16_matmul_workspace_bytes(64, 4096, 7168) == 0


def ffn(x=P, idx=P, probs=P, w1=P, s1=P, w2=P, s2=P, out=P, m=4, k=64, top_k=2, experts=8, n=32, fmt=E2M1, group=32, dtype=1, workspace=512, nbytes=None):
    L = _abi.lib()
    if nbytes is None:
        nbytes = L.cch_moe_ffn_w4a16_workspace_bytes(m, k, top_k, experts, n)
    return L.cch_moe_ffn_w4a16(x, idx, probs, w1, s1, None, w2, s2, None, out, m, k, top_k, experts, n, fmt, group, dtype, workspace, nbytes, None)


def test_moe_ffn_w4a16_arguments():
    L = _abi.lib()
    rejected(ffn(m=-1), "cch_moe_ffn_w4a16", "shape")
    rejected(ffn(m=BIG), "shape")
    rejected(ffn(k=(1 << 25) + 1), "shape")
    rejected(ffn(n=(1 << 25) + 2), "shape")
    rejected(ffn(m=1 << 29, top_k=8), "routes")
    rejected(ffn(n=33), "even")
    rejected(ffn(top_k=0), "top_k")
    rejected(ffn(top_k=9), "top_k")
    rejected(ffn(experts=0), "num_experts")
    rejected(ffn(experts=1025), "num_experts")
    rejected(ffn(fmt=1), "format 1")
    rejected(ffn(fmt=INT4, group=16), "group_size 16")
    rejected(ffn(dtype=3), "type 3")
    for missing in ("x", "idx", "probs", "w1", "s1", "w2", "s2", "out"):
        rejected(ffn(**{missing: None}), "null")
    rejected(ffn(workspace=None), "workspace")
    rejected(ffn(workspace=256), "512-byte boundary")
    rejected(ffn(nbytes=16), "workspace of 16 bytes")
    assert ffn(m=0, x=None, workspace=None) == _abi.OK
    assert L.cch_moe_ffn_w4a16_workspace_bytes(-1, 64, 2, 8, 32) == 0 and L.cch_moe_ffn_w4a16_workspace_bytes(4, 64, 0, 8, 32) == 0
