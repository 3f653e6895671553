"""w4a16_matmul and moe_ffn_w4a16 against the formulas in 64 bits.

Tolerances.  A result is rounded once to its type: half a unit, 2^-8 (bf16) or 2^-11 (half) of it.  Before that it is an fp32 sum: a
kernel may carry a code's distance from any integer up to 31, so with S = sum |x| (31 + |code - zero|) |scale| and no more than K / 32 + 64 roundings of
2^-24 one after the other, it is off by at most that much of S.  The block rounds its activation to 16 bits in between, half a unit of each element, which the
down projection carries along."""
import math

import pytest
import torch

import catccos_amd as cc

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def weights(gen, lead, k, fmt, group, zeros, dtype):
    """Codes, scales and zero points, every code and zero point used; scales such that a row's product is about one."""
    codes = torch.randint(0, 256, tuple(lead) + ((k + 1) // 2,), generator=gen, dtype=torch.uint8)
    if fmt == "e2m1":
        s = torch.randint(118, 126, tuple(lead) + (cc.scale_cols(k),), generator=gen, dtype=torch.uint8)
        return codes.cuda(), s.cuda(), None
    groups = (k + group - 1) // group
    s = ((torch.rand(tuple(lead) + (groups,), generator=gen) + 0.5) * 0.25 * max(k, 1) ** -0.5).to(dtype)
    z = torch.randint(0, 16, tuple(lead) + (groups,), generator=gen, dtype=torch.uint8) if zeros else None
    return codes.cuda(), s.cuda(), None if z is None else z.cuda()


def dense(w, k, fmt, group):
    """The weights' values in 64 bits, and the magnitudes that bound the sums' rounding."""
    codes, s, z = w
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., :k].long()
    per = 32 if fmt == "e2m1" else group
    at = torch.arange(k, device=codes.device) // per
    if fmt == "e2m1":
        scale = torch.exp2(s.double() - 127)[..., at]
        v = E2M1.to(codes.device)[q]
        return v * scale, v.abs() * scale
    scale = s.double()[..., at]
    v = q.double() - (8 if z is None else z.double()[..., at])
    return v * scale, (31 + v.abs()) * scale.abs()


def activations(gen, m, k, dtype):
    return (torch.randn(m, k, generator=gen) * torch.exp(0.5 * torch.randn(k, generator=gen))).to(dtype).cuda()


def check_product(x, w, fmt, group):
    out = cc.w4a16_matmul(x, *w, fmt=fmt, group_size=group)
    k = x.shape[1]
    v, bound = dense(w, k, fmt, group)
    want, size = x.double() @ v.t(), x.double().abs() @ bound.t()
    assert out.dtype == x.dtype and out.shape == want.shape
    err = (out.double() - want).abs()
    bad = err > UNIT[x.dtype] * want.abs() + (k / 32 + 64) * 2.0 ** -24 * size
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float(err.max()))
    assert float((out.double() - want).norm()) <= (UNIT[x.dtype] + 1e-4) * float(want.norm())
    return out


KINDS = [("int4", 32, False), ("int4", 64, True), ("int4", 128, False), ("int4", 128, True), ("e2m1", 32, False)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt,group,zeros", KINDS)
@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (1, 16, 128), (1, 512, 2048), (2, 17, 96), (3, 100, 160), (5, 300, 1984), (8, 64, 512), (15, 65, 1024), (16, 40, 4128),
                                   (17, 48, 256), (31, 33, 640), (32, 128, 1024), (33, 72, 544), (61, 200, 1216), (64, 64, 2048), (65, 50, 320), (130, 24, 256),
                                   (1, 4096, 64), (4, 2, 8192)])
def test_product(m, n, k, fmt, group, zeros, dtype):
    gen = torch.Generator().manual_seed(m * n + k)
    check_product(activations(gen, m, k, dtype), weights(gen, (n,), k, fmt, group, zeros, dtype), fmt, group)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt,group,zeros", KINDS)
@pytest.mark.parametrize("m,n,k", [(1, 5, 1), (2, 7, 2), (3, 9, 31), (5, 20, 33), (7, 12, 65), (4, 30, 100), (2, 11, 129), (18, 6, 1001), (1, 3, 260)])
def test_any_k(m, n, k, fmt, group, zeros, dtype):
    gen = torch.Generator().manual_seed(m * n + k)
    check_product(activations(gen, m, k, dtype), weights(gen, (n,), k, fmt, group, zeros, dtype), fmt, group)


@pytest.mark.parametrize("fmt,group,zeros", KINDS)
@pytest.mark.parametrize("m", [1, 4, 16, 24, 64])
def test_large_products(m, fmt, group, zeros):
    gen = torch.Generator().manual_seed(m)
    check_product(activations(gen, m, 7168, torch.bfloat16), weights(gen, (4096,), 7168, fmt, group, zeros, torch.bfloat16), fmt, group)


def test_weights_past_two_gibibytes():
    # rows behind 2^31 bytes of codes: their offsets pass 32 bits
    n, k = 540_000, 8192
    codes = torch.full((n, k // 2), 0x88, dtype=torch.uint8, device="cuda")          # the code 8: weights of zero
    scales = torch.ones((n, k // 128), dtype=torch.bfloat16, device="cuda")
    codes[n - 3] = 0x99
    codes[n - 1, -1] = 0x0F
    x = torch.ones(2, k, dtype=torch.bfloat16, device="cuda")
    x[1] = -0.5
    out = cc.w4a16_matmul(x, codes, scales)
    assert out[0, n - 3] == k and out[1, n - 3] == -k / 2 and out[0, n - 1] == 7 - 8 and out[0, n - 2] == 0
    assert int((out[0] != 0).sum()) == 2


def test_every_code_and_scale_of_mxfp4():
    # one nonzero activation per row: the product is one weight, exactly representable in bf16 or rounded once
    k = 64
    codes = torch.arange(256, dtype=torch.uint8).repeat(4).view(32, 32).cuda()
    for e in (0, 1, 60, 127, 180, 253):
        s = torch.full((32, 2), e, dtype=torch.uint8, device="cuda")
        x = torch.zeros(64, k, dtype=torch.bfloat16, device="cuda")
        x.fill_diagonal_(1.0)
        got = cc.w4a16_matmul(x, codes, s, fmt="e2m1").double()
        w = dense((codes, s, None), k, "e2m1", 32)[0]
        w = torch.where(w.abs() > 3.4e38, w * math.inf, w)    # past the range of fp32 and bf16: an infinity, which times zero is NaN
        want = x.double() @ w.t()
        tiny = 2.0 ** -126                                    # smaller results may be flushed to zero
        ok = (got == want) | (got.isnan() & want.isnan()) | ((want.abs() < tiny) & (got.abs() < tiny))
        assert ok.all(), e
    s = torch.full((32, 2), 127, dtype=torch.uint8, device="cuda")
    s[3, 1] = 255                                             # E8M0's NaN
    out = cc.w4a16_matmul(torch.ones(2, k, dtype=torch.bfloat16, device="cuda"), codes, s, fmt="e2m1")
    assert out[:, 3].isnan().all() and out[:, [i for i in range(32) if i != 3]].isfinite().all()


def test_the_row_quantisers_output_is_taken_as_it_is():
    gen = torch.Generator().manual_seed(2)
    w = torch.randn(96, 320, generator=gen).to(torch.bfloat16).cuda()
    payload, scales = cc.mx_quant(w, "e2m1")
    x = activations(gen, 6, 320, torch.bfloat16)
    check_product(x, (payload, scales, None), "e2m1", 32)
    ragged = torch.randn(20, 97, generator=gen).to(torch.bfloat16).cuda()
    check_product(activations(gen, 3, 97, torch.bfloat16), cc.mx_quant(ragged, "e2m1") + (None,), "e2m1", 32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt,group,zeros", KINDS)
def test_nan_and_infinity_stay_in_their_rows(fmt, group, zeros, dtype):
    # an activation that is not finite shows in its own row of the result alone, also where tiles are shared
    gen = torch.Generator().manual_seed(5)
    for m in (4, 16, 20):
        x = activations(gen, m, 256, dtype)
        w = weights(gen, (80,), 256, fmt, group, zeros, dtype)
        clean = cc.w4a16_matmul(x, *w, fmt=fmt, group_size=group)
        x[1, 77] = math.nan
        x[2, 200] = math.inf
        out = cc.w4a16_matmul(x, *w, fmt=fmt, group_size=group)
        assert out[1].isnan().all() and not out[2].isfinite().any()
        rest = [i for i in range(m) if i not in (1, 2)]
        assert torch.equal(out[rest], clean[rest])


def test_strides_alignment_and_streams():
    gen = torch.Generator().manual_seed(6)
    w = weights(gen, (70,), 512, "int4", 128, True, torch.bfloat16)
    x = activations(gen, 9, 512, torch.bfloat16)
    want = cc.w4a16_matmul(x, *w)
    wide = torch.zeros(9, 1024, dtype=torch.bfloat16, device="cuda")
    wide[:, ::2] = x
    assert torch.equal(cc.w4a16_matmul(wide[:, ::2], *w), want)
    tall = tuple(torch.stack([t, t], 1)[:, 0] for t in w)        # rows of the weights apart
    assert torch.equal(cc.w4a16_matmul(x, *tall), want)
    def shifted(t, by):                                           # contiguous, off the 16-byte boundaries
        raw = torch.zeros(t.numel() + by, dtype=t.dtype, device="cuda")
        raw[by:] = t.flatten()
        return raw[by:].view(t.shape)
    for args in ((shifted(x, 1), *w), (x, shifted(w[0], 3), *w[1:]), (x, w[0], shifted(w[1], 1), w[2]), (x, *w[:2], shifted(w[2], 1))):
        got = cc.w4a16_matmul(*args)
        assert float((got.double() - want.double()).norm()) <= 2 * (2.0 ** -8 + 1e-4) * float(want.double().norm())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = cc.w4a16_matmul(x, *w)
    s.synchronize()
    assert torch.equal(other, want) and torch.equal(cc.w4a16_matmul(x, *w), want)


def test_empty_products():
    w = weights(torch.Generator().manual_seed(0), (8,), 64, "int4", 32, False, torch.bfloat16)
    assert cc.w4a16_matmul(torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"), *w, group_size=32).shape == (0, 8)
    none = tuple(t[:0] if t is not None else None for t in w)
    assert cc.w4a16_matmul(torch.ones(3, 64, dtype=torch.bfloat16, device="cuda"), *none, group_size=32).shape == (3, 0)
    empty = (torch.empty(8, 0, dtype=torch.uint8, device="cuda"), torch.empty(8, 0, dtype=torch.bfloat16, device="cuda"), None)
    assert (cc.w4a16_matmul(torch.empty(3, 0, dtype=torch.bfloat16, device="cuda"), *empty) == 0).all()


def reference_block(x, idx, probs, w1, w2, fmt, group):
    """The block in 64 bits, and the bound of its error before the last rounding."""
    k = x.shape[1]
    v1, b1 = dense(w1, k, fmt, group)
    n = v1.shape[1]
    v2, b2 = dense(w2, n // 2, fmt, group)
    unit = UNIT[x.dtype]
    out, tol = torch.zeros(x.shape, dtype=torch.float64, device=x.device), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for e in range(v1.shape[0]):
        t, j = (idx == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        xe = x[t].double()
        up = xe @ v1[e].t()
        g, u = up[:, :n // 2], up[:, n // 2:]
        off = (k / 32 + 64) * 2.0 ** -24 * (xe.abs() @ b1[e].t())
        h = torch.nn.functional.silu(g) * u
        # silu's slope is at most 1.1; exp and division in fp32 add a few roundings
        dh = 1.1 * off[:, :n // 2] * u.abs() + torch.nn.functional.silu(g).abs() * off[:, n // 2:] + (unit + 2.0 ** -20) * h.abs() + 2.0 ** -25
        p = probs[t, j].double().unsqueeze(1)
        out.index_add_(0, t, p * (h @ v2[e].t()))
        tol.index_add_(0, t, p.abs() * (dh @ v2[e].abs().t() + (n / 64 + 80) * 2.0 ** -24 * ((h.abs() + dh) @ b2[e].t())))
    return out, tol


def check_block(x, idx, probs, w1, w2, fmt, group):
    out = cc.moe_ffn_w4a16(x, idx, probs, *w1, *w2, fmt=fmt, group_size=group)
    want, tol = reference_block(x, idx, probs, w1, w2, fmt, group)
    err = (out.double() - want).abs()
    assert out.dtype == x.dtype and (err <= tol + UNIT[x.dtype] * (want.abs() + tol)).all(), float((err / (tol + 1e-9)).max())
    assert float(err.norm()) <= (2.2 * UNIT[x.dtype] + 2e-4) * float(want.norm())
    return out


def block(seed, m, k, n, e, top_k, fmt, group, zeros, dtype):
    gen = torch.Generator().manual_seed(seed)
    x = activations(gen, m, k, dtype)
    w1, w2 = weights(gen, (e, n), k, fmt, group, zeros, dtype), weights(gen, (e, k), n // 2, fmt, group, zeros, dtype)
    scores = torch.rand(m, e, generator=gen) + torch.rand(e, generator=gen)
    top = scores.topk(top_k, dim=1)
    probs = (top.values / top.values.sum(1, keepdim=True)).cuda()
    return x, top.indices.int().cuda(), probs, w1, w2


@pytest.mark.parametrize("fmt,group,zeros", KINDS)
@pytest.mark.parametrize("m,k,n,e,top_k,dtype", [(1, 128, 64, 1, 1, torch.bfloat16), (1, 256, 128, 8, 4, torch.float16), (3, 192, 320, 5, 2, torch.bfloat16),
                                                 (17, 512, 256, 4, 3, torch.float16), (40, 256, 512, 16, 6, torch.bfloat16), (70, 320, 192, 3, 1, torch.bfloat16),
                                                 (33, 1024, 512, 64, 8, torch.bfloat16), (100, 96, 64, 2, 2, torch.float16), (5, 100, 30, 7, 3, torch.bfloat16),
                                                 (2, 63, 66, 4, 2, torch.float16)])
def test_block(m, k, n, e, top_k, dtype, fmt, group, zeros):
    x, idx, probs, w1, w2 = block(m + k, m, k, n, e, top_k, fmt, group, zeros, dtype)
    check_block(x, idx, probs, w1, w2, fmt, group)


@pytest.mark.parametrize("m", [1, 64])
def test_large_block(m):
    check_block(*block(m, m, 2048, 2048, 16, 6, "int4", 128, False, torch.bfloat16), "int4", 128)


def test_dropped_routes_one_expert_for_all_and_the_same_one_twice():
    x, idx, probs, w1, w2 = block(3, 24, 256, 128, 6, 3, "int4", 64, True, torch.bfloat16)
    idx[0] = -1                       # no route at all: a row of zeros
    idx[1, 1] = -1
    idx[2, 0] = 6
    idx[3, 2] = 1 << 30
    out = check_block(x, idx, probs, w1, w2, "int4", 64)
    assert (out[0] == 0).all()
    same = torch.full_like(idx, 4)    # every route of every token
    check_block(x, same, probs, w1, w2, "int4", 64)
    assert torch.equal(cc.moe_ffn_w4a16(x, same, probs, *w1, *w2, group_size=64), cc.moe_ffn_w4a16(x, same, probs, *w1, *w2, group_size=64))
    none = torch.full_like(idx, -1)
    assert (cc.moe_ffn_w4a16(x, none, probs, *w1, *w2, group_size=64) == 0).all()


def test_a_dropped_tokens_values_go_nowhere():
    x, idx, probs, w1, w2 = block(4, 20, 256, 128, 4, 2, "int4", 128, False, torch.bfloat16)
    clean = cc.moe_ffn_w4a16(x, idx, probs, *w1, *w2)
    x[5] = math.nan
    idx[5] = -1
    probs[5] = math.nan
    out = cc.moe_ffn_w4a16(x, idx, probs, *w1, *w2)
    assert (out[5] == 0).all()
    rest = [i for i in range(20) if i != 5]
    assert torch.equal(out[rest], clean[rest])


def test_many_routes():
    # more routes than any table in LDS holds, a skewed choice of experts
    x, idx, probs, w1, w2 = block(5, 3000, 64, 64, 9, 8, "int4", 32, False, torch.bfloat16)
    check_block(x, idx, probs, w1, w2, "int4", 32)


def test_gate_and_block_together():
    gen = torch.Generator().manual_seed(8)
    x, _, _, w1, w2 = block(8, 30, 256, 128, 8, 2, "e2m1", 32, False, torch.bfloat16)
    gate = (torch.randn(8, 256, generator=gen) / 16).cuda()
    mask = torch.ones(30, dtype=torch.bool, device="cuda")
    mask[7:11] = False
    probs, idx = cc.moe_router(x.float() @ gate.t(), 2, token_mask=mask)
    out = check_block(x, idx, probs, w1, w2, "e2m1", 32)
    assert (out[7:11] == 0).all() and (out[:7] != 0).any()


def test_empty_block():
    x, idx, probs, w1, w2 = block(1, 4, 64, 32, 2, 1, "int4", 32, False, torch.bfloat16)
    assert cc.moe_ffn_w4a16(x[:0], idx[:0], probs[:0], *w1, *w2, group_size=32).shape == (0, 64)
    nothing = lambda w, rows, cols: (w[0][:, :rows, :cols // 2], w[1][:, :rows, :(cols + 31) // 32], None)   # noqa: E731
    assert (cc.moe_ffn_w4a16(x, idx, probs, *nothing(w1, 0, 64), *nothing(w2, 64, 0), group_size=32) == 0).all()


def test_block_strides_alignment_and_streams():
    x, idx, probs, w1, w2 = block(6, 12, 256, 128, 4, 2, "int4", 128, True, torch.float16)
    want = cc.moe_ffn_w4a16(x, idx, probs, *w1, *w2)
    wide = torch.stack([x, x], 1)[:, 0]
    pair = torch.stack([idx, idx], 2)[..., 0]
    assert torch.equal(cc.moe_ffn_w4a16(wide, pair, torch.stack([probs, probs], 2)[..., 0], *w1, *w2), want)
    raw = torch.zeros(w1[0].numel() + 5, dtype=torch.uint8, device="cuda")
    raw[5:] = w1[0].flatten()
    got = cc.moe_ffn_w4a16(x, idx, probs, raw[5:].view(w1[0].shape), *w1[1:], *w2)
    assert float((got.double() - want.double()).norm()) <= 5e-3 * float(want.double().norm())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = cc.moe_ffn_w4a16(x, idx, probs, *w1, *w2)
    s.synchronize()
    assert torch.equal(other, want)


def test_refusals():
    gen = torch.Generator().manual_seed(0)
    x = activations(gen, 2, 64, torch.bfloat16)
    w, s, z = weights(gen, (8,), 64, "int4", 32, True, torch.bfloat16)
    ok = lambda *a, **kw: cc.w4a16_matmul(*a, **{"group_size": 32, **kw})   # noqa: E731
    for bad in (lambda: ok(x.cpu(), w, s), lambda: ok(x, w.cpu(), s), lambda: ok(x.float(), w, s), lambda: ok(x[0], w, s), lambda: ok(x, w, s.float()),
                lambda: ok(x, w, s.half()), lambda: ok(x, w, s, z.int()), lambda: ok(x, w, s, z[:, :1]), lambda: ok(x, w, s, group_size=48),
                lambda: ok(x, w, s, group_size=64), lambda: ok(x, w[:, :31], s), lambda: ok(x, w, s[:7]), lambda: ok(x, w, s, fmt="int8"),
                lambda: ok(x, w, s, fmt="e2m1"), lambda: ok(x, w, s.view(torch.uint8)[:, :2], z, fmt="e2m1"), lambda: ok(x, w.to(torch.int8), s)):
        with pytest.raises(ValueError):
            bad()
    x, idx, probs, w1, w2 = block(1, 4, 64, 32, 3, 2, "int4", 32, True, torch.bfloat16)
    ffn = lambda *a: cc.moe_ffn_w4a16(*a, group_size=32)   # noqa: E731
    for bad in (lambda: ffn(x, idx.long(), probs, *w1, *w2), lambda: ffn(x, idx, probs.half(), *w1, *w2), lambda: ffn(x, idx[:3], probs, *w1, *w2),
                lambda: ffn(x, idx, probs[:, :1], *w1, *w2), lambda: ffn(x, idx, probs, *w2, *w1), lambda: ffn(x, idx, probs, *w1, *(t[:2] for t in w2)),
                lambda: ffn(x, idx, probs, *(t[:, :31] for t in w1), *w2), lambda: ffn(x, idx.repeat(1, 5), probs.repeat(1, 5), *w1, *w2),
                lambda: ffn(x, idx.cpu(), probs, *w1, *w2)):
        with pytest.raises(ValueError):
            bad()
