"""One mixture-of-experts layer from its gate's training to its decode steps, on one GPU with synthetic data:

  * a gate learns which experts suit a token (moe_router, differentiable) while the balance and z loss (moe_balance_loss) keep the experts' loads even;
  * the experts' and the output projection's weights are packed to 4 bits, integers in groups or MXFP4;
  * a decode step - gate, 4-bit experts (moe_ffn_w4a16), 4-bit output projection (w4a16_matmul) - is recorded as one HIP graph, replayed, and compared with the
    eager step (the same bits) and with fp32 products of the unpacked weights.

    python -m catccos_amd.run_moe_w4
    python -m catccos_amd.run_moe_w4 --fmt e2m1 --batch 32 --scoring sigmoid

Exit status 1 if the loads did not even out or a decode step is wrong.
"""
import argparse
import sys

import torch

import catccos_amd as cc


def train_gate(a, gen):
    """The gate [E, k] (fp32), trained on `tokens` tokens of eight kinds, most of one; returns it with the load of the busiest expert before and after."""
    kinds = torch.randn(8, a.k, generator=gen, device="cuda")
    which = torch.multinomial(torch.tensor([8.0, 4, 2, 1, 1, 1, 1, 1], device="cuda"), a.tokens, replacement=True, generator=gen)
    x = kinds[which] + 0.5 * torch.randn(a.tokens, a.k, generator=gen, device="cuda")
    suits = torch.randn(8, a.experts, generator=gen, device="cuda")[which]       # what an expert is worth to a token
    gate = (torch.randn(a.experts, a.k, generator=gen, device="cuda") / a.k ** 0.5).requires_grad_()
    opt = torch.optim.Adam([gate], lr=1e-2 / a.k ** 0.5)
    even, loads = a.tokens * a.topk / a.experts, []
    for step in range(a.steps):
        logits = x @ gate.t()
        probs, idx = cc.moe_router(logits, a.topk, scoring=a.scoring)
        balance, counts, _ = cc.moe_balance_loss(logits, idx, coef=a.coef, z_coef=1e-4, scoring=a.scoring)
        worth = (probs * suits.gather(1, idx.long())).sum(1).mean()
        opt.zero_grad(set_to_none=True)
        (balance - worth).backward()
        opt.step()
        loads.append(float(counts.max()) / even)
        if step % 20 == 0 or step == a.steps - 1:
            print("  step %3d  worth %6.3f  balance + z loss %6.4f  busiest expert %.2f x the even load" % (step, worth.item(), balance.item(), loads[-1]), flush=True)
    return gate.detach(), loads[0], loads[-1]


def pack(w, fmt, group, dtype):
    """Weights [..., K] to (codes, scales, zeros) and what these stand for, fp32."""
    if fmt == "e2m1":
        flat = w.reshape(-1, w.shape[-1]).to(torch.bfloat16)
        codes, scales = cc.mx_quant(flat, "e2m1")
        values = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
        q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
        back = values[q] * torch.exp2(scales.float() - 127).repeat_interleave(32, 1)[:, :w.shape[-1]]
        return (codes.view(*w.shape[:-1], -1), scales.view(*w.shape[:-1], -1), None), back.view(w.shape)
    g = w.unflatten(-1, (-1, group))
    scales = (g.amax(-1) - g.amin(-1)).div(15).clamp_min(1e-8).to(dtype)
    zeros = (-g.amin(-1) / scales.float()).round().clamp(0, 15)
    q = (g / scales.float().unsqueeze(-1) + zeros.unsqueeze(-1)).round().clamp(0, 15)
    back = ((q - zeros.unsqueeze(-1)) * scales.float().unsqueeze(-1)).flatten(-2)
    q = q.flatten(-2).to(torch.uint8)
    return (q[..., ::2] | q[..., 1::2] << 4, scales, zeros.to(torch.uint8)), back


def decode(a, gate, gen):
    """Replays of the recorded step; returns the largest error relative to the fp32 products' norm and whether replays and eager steps agree to the bit."""
    dtype = torch.float16 if a.half else torch.bfloat16
    def new(*shape):
        return torch.randn(*shape, generator=gen, device="cuda") / shape[-1] ** 0.5
    w1, v1 = pack(new(a.experts, a.n, a.k), a.fmt, a.group, dtype)
    w2, v2 = pack(new(a.experts, a.k, a.n // 2), a.fmt, a.group, dtype)
    wo, vo = pack(new(a.vocab, a.k), a.fmt, a.group, dtype)
    x = torch.randn(a.batch, a.k, generator=gen, device="cuda").to(dtype)
    gate16 = gate.to(dtype)
    kw = {"fmt": a.fmt, "group_size": a.group}

    def step():
        probs, idx = cc.moe_router(x @ gate16.t(), a.topk, scoring=a.scoring)
        y = x + cc.moe_ffn_w4a16(x, idx, probs, *w1, *w2, **kw)
        return idx, probs, y, cc.w4a16_matmul(y, *wo, **kw)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    same, worst = True, 0.0
    for _ in range(3):
        x.copy_(torch.randn(a.batch, a.k, generator=gen, device="cuda"))
        for t in held:
            t.zero_()
        graph.replay()
        eager = step()
        same = same and all(torch.equal(h, e) for h, e in zip(held, eager))
        idx, probs, y, out = eager
        want = x.float()
        for j in range(a.topk):
            up = torch.bmm(v1[idx[:, j].long()], x.float().unsqueeze(2)).squeeze(2)
            h = torch.nn.functional.silu(up[:, :a.n // 2]) * up[:, a.n // 2:]
            want = want + probs[:, j:j + 1] * torch.bmm(v2[idx[:, j].long()], h.unsqueeze(2)).squeeze(2)
        for got, ref in ((y, want), (out, y.float() @ vo.t())):
            worst = max(worst, float((got.float() - ref).norm() / ref.norm()))
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    start.record()
    for _ in range(a.replays):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    print("  %d tokens a step: %.1f us, error %.4f of the fp32 products" % (a.batch, start.elapsed_time(end) * 1e3 / a.replays, worst), flush=True)
    return worst, same


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=4096, help="tokens of a training step")
    ap.add_argument("--steps", type=int, default=100)
    ap.add_argument("--coef", type=float, default=4.0, help="weight of the balance loss")
    ap.add_argument("--k", type=int, default=2048, help="width of the layer, a multiple of the group")
    ap.add_argument("--n", type=int, default=1024, help="columns of an expert's up projection, gate and up halves; half of it a multiple of the group")
    ap.add_argument("--experts", type=int, default=16)
    ap.add_argument("--topk", type=int, default=4)
    ap.add_argument("--scoring", choices=["softmax", "sigmoid"], default="softmax")
    ap.add_argument("--vocab", type=int, default=8192, help="rows of the output projection")
    ap.add_argument("--batch", type=int, default=8, help="tokens of a decode step")
    ap.add_argument("--fmt", choices=["int4", "e2m1"], default="int4")
    ap.add_argument("--group", type=int, choices=[32, 64, 128], default=128)
    ap.add_argument("--half", action="store_true", help="half activations instead of bf16")
    ap.add_argument("--replays", type=int, default=200)
    a = ap.parse_args(argv)
    gen = torch.Generator(device="cuda").manual_seed(0)
    print("gate: %d experts, %d routes a token, %s scores" % (a.experts, a.topk, a.scoring), flush=True)
    gate, before, after = train_gate(a, gen)
    print("decode: %s weights, %s activations" % (a.fmt, "half" if a.half else "bf16"), flush=True)
    worst, same = decode(a, gate, gen)
    # roundings to 16 bits, of the activation between the products and of the results: each 2^-8 at most, a third of it on average
    ok = after < before and worst < 2.0 ** -7 and same
    print("ok" if ok else "FAILED: loads %.2f -> %.2f, error %.4f, replays %s" % (before, after, worst, "agree" if same else "differ"))
    return 0 if ok else 1


if __name__ == "__main__":
    sys.exit(main())
