"""What a mixture-of-experts model asks for around the expert products, and the products of a decode step with 4-bit weights.

Four operators, each called as a user's program calls it:

    router    scores of the gate's logits, the top-k experts and their weights; in training the logits' gradient too
    balance   the balance loss, the z loss and the tokens per expert of a batch or of each of its sequences, and the logits' gradient
    w4        a linear layer of a decode step: bf16 or half activations, 4-bit weights with a scale per group along K
    moe_w4    the mixture-of-experts feed-forward of a decode step with such weights, routing to combine

`run` computes them from the formulas with elementary torch operations in 32 bits, or, where `own` is true, calls the package.
Sizes of layers are those of this repository's configurations and shape lists, and in draw() others of the same kind."""
import math

import torch

own = False


def listed():
    return [
        # the gate of a decode step of 64 sequences, 6 of 16 experts each: the smallest call there is
        {"name": "router-decode", "kind": "router", "m": 64, "e": 16, "top_k": 6, "dtype": "f32", "scoring": "softmax", "renorm": True, "scale": 1.0,
         "pad": False, "off": False, "backward": False},
        # the gate of a training step over 16384 tokens, 8 of 64 experts, with its gradient
        {"name": "router-train", "kind": "router", "m": 16384, "e": 64, "top_k": 8, "dtype": "bf16", "scoring": "softmax", "renorm": False, "scale": 1.0,
         "pad": False, "off": False, "backward": True},
        # a ragged batch with padding and one expert out of service: sigmoid scores, renormalised and scaled, with the gradient
        {"name": "router-sigmoid", "kind": "router", "m": 4099, "e": 256, "top_k": 8, "dtype": "f32", "scoring": "sigmoid", "renorm": True, "scale": 2.5,
         "pad": True, "off": True, "backward": True},
        # the loss of a small batch, 6 of 16 experts
        {"name": "balance-small", "kind": "balance", "m": 512, "e": 16, "top_k": 6, "dtype": "f32", "scoring": "softmax", "z": 1e-3, "pad": False, "seqs": 0},
        # the loss of a large ragged batch taken per sequence, sigmoid scores, padding between
        {"name": "balance-sequences", "kind": "balance", "m": 16384, "e": 256, "top_k": 8, "dtype": "bf16", "scoring": "sigmoid", "z": 0.0, "pad": True, "seqs": 13},
        # one token through a dense layer of 4-bit integers, groups of 128: where latency counts
        {"name": "w4-one", "kind": "w4", "m": 1, "k": 7168, "n": 4096, "fmt": "int4", "group": 128, "zeros": False, "half": False},
        # a decode step of 16 sequences, MXFP4 weights
        {"name": "w4-mx-16", "kind": "w4", "m": 16, "k": 2048, "n": 7168, "fmt": "e2m1", "group": 32, "zeros": False, "half": False},
        # a layer none of whose sizes is a power of two, small groups with zero points, half activations
        {"name": "w4-ragged", "kind": "w4", "m": 5, "k": 1984, "n": 3000, "fmt": "int4", "group": 32, "zeros": True, "half": True},
        # 61 sequences against the widest layer there is, an output projection
        {"name": "w4-wide-61", "kind": "w4", "m": 61, "k": 7168, "n": 32768, "fmt": "int4", "group": 64, "zeros": True, "half": False},
        # one token through the mixture-of-experts block, 6 of 16 experts
        {"name": "moe-w4-one", "kind": "moe_w4", "m": 1, "k": 7168, "n": 4096, "e": 16, "top_k": 6, "fmt": "int4", "group": 128, "zeros": False, "half": False},
        # 64 tokens through the same block, MXFP4 weights: every expert is read
        {"name": "moe-w4-64", "kind": "moe_w4", "m": 64, "k": 7168, "n": 4096, "e": 16, "top_k": 6, "fmt": "e2m1", "group": 32, "zeros": False, "half": False},
        # many small experts, few tokens for each, zero points
        {"name": "moe-w4-small", "kind": "moe_w4", "m": 33, "k": 2048, "n": 1024, "e": 64, "top_k": 8, "fmt": "int4", "group": 64, "zeros": True, "half": False},
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    v = min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return v + (v == 3072)


def _dim(rng, lo, hi, unit):
    """A layer's size: some a power of two, the others a multiple of 512, 128 or `unit`."""
    v = _log(rng, lo, hi)
    u = rng.choice([0, 512, 128, unit])
    v = 1 << v.bit_length() - 1 if u == 0 else max(lo, v // u * u)
    return v + 128 if v % 3072 == 0 else v


def draw(rng):
    while True:
        kind = rng.choice(["router", "balance", "w4", "w4", "moe_w4", "moe_w4"])
        c = {"kind": kind}
        if kind in ("router", "balance"):
            c.update(m=_log(rng, 1, 16384), e=rng.choice([8, 16, 20, 32, 60, 64, 72, 128, 160, 256]))
            c.update(top_k=rng.choice([1, 2, 4, 6, 8]), dtype=rng.choice(["f32", "f32", "bf16", "f16"]), scoring=rng.choice(["softmax", "sigmoid"]),
                     pad=rng.random() < 0.3)
            if kind == "router":
                c.update(renorm=rng.random() < 0.5, scale=rng.choice([1.0, 1.0, 2.5]), off=rng.random() < 0.3 and c["top_k"] < c["e"], backward=rng.random() < 0.6)
            else:
                c.update(z=rng.choice([0.0, 1e-3]), seqs=rng.choice([0, 0, 1, 4, 13, 40]))
            return c
        c.update(m=_log(rng, 1, 128), k=_dim(rng, 512, 8192, 32), fmt=rng.choice(["int4", "int4", "e2m1"]), half=rng.random() < 0.3)
        c["group"] = 32 if c["fmt"] == "e2m1" else rng.choice([32, 64, 128, 128])
        c["zeros"] = c["fmt"] == "int4" and rng.random() < 0.5
        if kind == "w4":
            c["n"] = _dim(rng, 512, 32768, 8)
            if c["m"] * c["k"] * c["n"] <= 61 * 7168 * 32768:
                return c
            continue
        c["n"] = max(512, _dim(rng, 512, 8192, 64) // 64 * 64)        # gate and up halves
        c["e"] = rng.choice([4, 8, 16, 32, 64])
        c["top_k"] = rng.choice([t for t in (1, 2, 4, 6, 8) if t <= c["e"]])
        if c["e"] * c["k"] * c["n"] <= 16 * 7168 * 4096 and c["m"] * c["top_k"] * c["k"] * c["n"] <= 64 * 6 * 7168 * 4096:
            return c


_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _code(gen, shape, c):
    """Weights of variance 1/K as a checkpoint holds them: packed codes [..., K/2], scales, zero points or None."""
    k, g = shape[-1], c["group"]
    x = torch.randn(shape, device="cuda", generator=gen) * k ** -0.5
    x = torch.nn.functional.pad(x, (0, -k % g)).unflatten(-1, (-1, g))
    z = None
    if c["fmt"] == "e2m1":
        e = torch.floor(torch.log2(x.abs().amax(-1).clamp_min(1e-30))) - 2
        v = x / torch.exp2(e).unsqueeze(-1)
        edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
        q = torch.bucketize(v.abs(), edges, out_int32=True) + 8 * (v < 0).int()
        s = (e + 127).to(torch.uint8)
        s = torch.nn.functional.pad(s, (0, s.shape[-1] % 2), value=127)
    elif c["zeros"]:
        lo, hi = x.amin(-1).clamp_max(0), x.amax(-1).clamp_min(0)
        s = ((hi - lo) / 15).clamp_min(1e-6).to(torch.float16 if c["half"] else torch.bfloat16)
        z = torch.round(-lo / s.float()).clamp(0, 15).to(torch.uint8)
        q = (torch.round(x / s.float().unsqueeze(-1)) + z.unsqueeze(-1)).clamp(0, 15).int()
    else:
        s = (x.abs().amax(-1) / 7).clamp_min(1e-6).to(torch.float16 if c["half"] else torch.bfloat16)
        q = (torch.round(x / s.float().unsqueeze(-1)) + 8).clamp(0, 15).int()
    q = q.flatten(-2)[..., :k]
    return (q[..., 0::2] | q[..., 1::2] << 4).to(torch.uint8).contiguous(), s.contiguous(), z


def _activations(gen, m, k, half):
    """Activations as a normalisation leaves them: unit variance, a few channels an order of magnitude larger."""
    gain = torch.exp(0.5 * torch.randn(k, device="cuda", generator=gen))
    return (torch.randn(m, k, device="cuda", generator=gen) * gain).to(torch.float16 if half else torch.bfloat16)


def _logits(gen, m, e):
    """A gate's logits: some experts liked more than others by all tokens, and each token's own likes."""
    return 1.5 * torch.randn(m, e, device="cuda", generator=gen) + 0.7 * torch.randn(e, device="cuda", generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    c = dict(case)
    kind, m = c["kind"], c["m"]
    s = {"case": c}
    if kind in ("router", "balance"):
        e, k = c["e"], c["top_k"]
        loss_scale = 65536.0 if c["dtype"] == "f16" else 1.0   # as training in halves has it
        logits = _logits(gen, m, e)
        if c.get("off"):
            logits[:, int(torch.randint(e, (1,), device="cuda", generator=gen))] = -math.inf
        s["logits"] = logits.to(_TYPES[c["dtype"]])
        s["mask"] = torch.rand(m, device="cuda", generator=gen) < 0.9 if c["pad"] else None
        if kind == "router":
            s["grad"] = torch.randn(m, k, device="cuda", generator=gen) / m * loss_scale
        else:
            idx = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32)
            s["idx"] = idx.masked_fill(~s["mask"].unsqueeze(1), -1) if c["pad"] else idx
            s["grad"] = torch.full((), loss_scale, device="cuda")
            s["offsets"] = None
            if c["seqs"]:
                cuts = torch.randint(0, m + 1, (c["seqs"] - 1,), device="cuda", generator=gen).sort().values
                s["offsets"] = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), m)]).to(torch.int32)
        return s
    n, k = c["n"], c["k"]
    s["x"] = _activations(gen, m, k, c["half"])
    if kind == "w4":
        s["w"] = _code(gen, (n, k), c)
        return s
    e = c["e"]
    s["w1"], s["w2"] = ([None, None, None], [None, None, None])
    for at, rows, cols in (("w1", n, k), ("w2", k, n // 2)):
        parts = [_code(gen, (rows, cols), c) for _ in range(e)]
        s[at] = tuple(torch.stack([p[i] for p in parts]) if parts[0][i] is not None else None for i in range(3))
    top = _logits(gen, m, e).softmax(1).topk(c["top_k"], dim=1)
    s["idx"] = top.indices.to(torch.int32)
    s["probs"] = top.values / top.values.sum(1, keepdim=True)
    return s


def _plain_scores(l, scoring):
    if scoring == "sigmoid":
        return 1 / (1 + torch.exp(-l))
    x = torch.exp(l - l.amax(1, keepdim=True))
    return x / x.sum(1, keepdim=True)


def _plain_router(s, c):
    l = s["logits"].float()
    order = torch.sort(l, dim=1, descending=True, stable=True)
    idx = order.indices[:, :c["top_k"]]
    there = order.values[:, :c["top_k"]] > -math.inf
    if s["mask"] is not None:
        there = there & s["mask"].unsqueeze(1)
    scores = _plain_scores(l, c["scoring"])
    w = torch.where(there, scores.gather(1, idx), 0)
    total = w.sum(1, keepdim=True)
    probs = c["scale"] * w / torch.where(total > 0, total, 1) if c["renorm"] else c["scale"] * w
    out = {"probs": probs, "idx": torch.where(there, idx, -1).to(torch.int32)}
    if c["backward"]:
        g = s["grad"]
        if c["renorm"]:   # of the scores that were divided by their sum
            g = (g - (g * probs).sum(1, keepdim=True) / c["scale"]) / torch.where(total > 0, total, 1)
        g = torch.zeros_like(l).scatter_(1, idx, torch.where(there, c["scale"] * g, 0))
        d = scores * (g - (g * scores).sum(1, keepdim=True)) if c["scoring"] == "softmax" else g * scores * (1 - scores)
        out["grad"] = d.to(s["logits"].dtype)
    return out


def _plain_balance(s, c):
    l = s["logits"].float()
    m, e = l.shape
    counted = (s["mask"] if s["mask"] is not None else torch.ones(m, dtype=torch.bool, device=l.device)).float()
    if s["offsets"] is None:
        member = counted.unsqueeze(1)                                                            # [m, sequences]
    else:
        t = torch.arange(m, device=l.device).unsqueeze(1)
        member = ((t >= s["offsets"][:-1]) & (t < s["offsets"][1:])).float() * counted.unsqueeze(1)
    tokens = member.sum(0)
    routed = torch.zeros(m, e + 1, device=l.device).scatter_add_(1, torch.where(s["idx"] >= 0, s["idx"], e).long(), torch.ones_like(s["idx"], dtype=torch.float32))[:, :e]
    counts = member.t() @ routed
    share = e / c["top_k"] * counts / tokens.clamp_min(1).unsqueeze(1)
    sc = _plain_scores(l, c["scoring"])
    p = sc / sc.sum(1, keepdim=True)
    mean = member.t() @ p / tokens.clamp_min(1).unsqueeze(1)
    alive = (tokens > 0).sum().clamp_min(1)
    top = l.amax(1, keepdim=True)
    ex = torch.exp(l - top)
    lse = torch.log(ex.sum(1, keepdim=True)) + top
    total = tokens.sum().clamp_min(1)
    inside = member.sum(1, keepdim=True)
    loss = 0.01 * (share * mean).sum() / alive + c["z"] * (inside * lse * lse).sum() / total
    v = (member / tokens.clamp_min(1)) @ share * (0.01 / alive)
    d = p * (v - (v * p).sum(1, keepdim=True))
    if c["scoring"] == "sigmoid":
        d = d * (1 - sc)
    d = s["grad"] * (d + c["z"] * 2 / total * inside * lse * ex / ex.sum(1, keepdim=True))
    counts = counts.to(torch.int32)
    return {"loss": loss, "counts": counts if s["offsets"] is not None else counts[0], "tokens": tokens.to(torch.int32), "grad": d.to(s["logits"].dtype)}


def _plain_weights(w, c, k):
    q, s, z = w
    q = torch.stack([q & 15, q >> 4], -1).flatten(-2)
    if c["fmt"] == "e2m1":
        v = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=q.device)[q.int()]
        s = torch.exp2(s.float() - 127)
    else:
        v = q.float() - (8 if z is None else z.float().repeat_interleave(c["group"], -1)[..., :k])
        s = s.float()
    return v * s.repeat_interleave(c["group"], -1)[..., :k]


def _plain_w4(s, c):
    return (s["x"].float() @ _plain_weights(s["w"], c, c["k"]).t()).to(s["x"].dtype)


def _plain_moe(s, c):
    x = s["x"].float()
    up = torch.matmul(x.unsqueeze(0), _plain_weights(s["w1"], c, c["k"]).transpose(1, 2).contiguous())         # [e, m, n]
    gate, lin = up.chunk(2, dim=2)
    y = torch.matmul(gate / (1 + torch.exp(-gate)) * lin, _plain_weights(s["w2"], c, c["n"] // 2).transpose(1, 2).contiguous())
    share = torch.zeros(c["m"], c["e"], device=x.device).scatter_(1, s["idx"].long(), s["probs"])
    return (share.t().unsqueeze(2) * y).sum(0).to(s["x"].dtype)


def run(state):
    c = state["case"]
    kind = c["kind"]
    if not own:
        return {"router": _plain_router, "balance": _plain_balance, "w4": _plain_w4, "moe_w4": _plain_moe}[kind](state, c)
    import catccos_amd as cc
    s = state
    if kind == "router":
        probs, idx = cc.moe_router(s["logits"], c["top_k"], scoring=c["scoring"], renormalize=c["renorm"], scale=c["scale"], token_mask=s["mask"])
        out = {"probs": probs, "idx": idx}
        if c["backward"]:
            out["grad"] = cc.moe_router_backward(s["grad"], s["logits"], idx, scoring=c["scoring"], renormalize=c["renorm"], scale=c["scale"])
        return out
    if kind == "balance":
        opt = {"coef": 0.01, "z_coef": c["z"], "scoring": c["scoring"], "token_mask": s["mask"], "seq_offsets": s["offsets"]}
        loss, counts, tokens = cc.moe_balance_loss(s["logits"], s["idx"], **opt)
        return {"loss": loss, "counts": counts, "tokens": tokens,
                "grad": cc.moe_balance_loss_backward(s["grad"], s["logits"], counts, tokens, c["top_k"], **opt)}
    if kind == "w4":
        return cc.w4a16_matmul(s["x"], *s["w"], fmt=c["fmt"], group_size=c["group"])
    return cc.moe_ffn_w4a16(s["x"], s["idx"], s["probs"], *s["w1"], *s["w2"], fmt=c["fmt"], group_size=c["group"])


def work(case):
    c = case
    m = c["m"]
    if c["kind"] in ("router", "balance"):
        size = 4 if c["dtype"] == "f32" else 2
        le, lk = m * c["e"], m * c["top_k"]
        if c["kind"] == "router":
            # logits in, weights and experts out; the gradient's pass reads the logits, the weights' gradient and the experts
            return {"bytes": le * size + 8 * lk + m * c["pad"] + ((2 * le * size + 8 * lk) if c["backward"] else 0), "flops": le * (10 if c["backward"] else 5)}
        return {"bytes": 3 * le * size + 4 * lk + 2 * m * c["pad"] + 4 * c["e"] * max(1, c["seqs"]) * 2, "flops": le * 20}
    per = 0.5 + (1 if c["fmt"] == "e2m1" else 2 + c["zeros"]) / c["group"]     # bytes of a weight
    k, n = c["k"], c["n"]
    if c["kind"] == "w4":
        return {"bytes": per * n * k + 2 * m * (n + k), "flops": 2.0 * m * n * k}
    read = c["e"] * (1 - (1 - c["top_k"] / c["e"]) ** m)                       # experts that some token names
    return {"bytes": per * 1.5 * n * k * read + 4 * m * k + 8 * m * c["top_k"], "flops": 3.0 * m * c["top_k"] * n * k}


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["kind"] in ("router", "balance"):
        l = s["logits"].double()
        m, e = l.shape
        use = s["mask"] if s["mask"] is not None else torch.ones(m, dtype=torch.bool, device=l.device)
        sm = torch.softmax(l, 1)
        sg = torch.sigmoid(l)
    if c["kind"] == "router":
        idx = torch.argsort(-l, dim=1, stable=True)[:, :c["top_k"]]
        scores = sm if c["scoring"] == "softmax" else sg
        chosen = scores.gather(1, idx)
        w = c["scale"] * (chosen / chosen.sum(1, keepdim=True) if c["renorm"] else chosen)
        out = {"probs": w * use.unsqueeze(1), "idx": None}
        if c["backward"]:
            g = s["grad"].double() * use.unsqueeze(1)
            if c["renorm"]:
                d = w * (g - (g * w).sum(1, keepdim=True) / c["scale"])
                if c["scoring"] == "sigmoid":
                    d = d * (1 - chosen)
                out["grad"] = torch.zeros_like(l).scatter(1, idx, d)
            elif c["scoring"] == "sigmoid":
                out["grad"] = torch.zeros_like(l).scatter(1, idx, g * w * (1 - chosen))
            else:
                out["grad"] = torch.zeros_like(l).scatter(1, idx, g * w) - sm * (g * w).sum(1, keepdim=True)
        return out
    if c["kind"] == "balance":
        p = sm if c["scoring"] == "softmax" else sg / sg.sum(1, keepdim=True)
        lse = torch.logsumexp(l, 1)
        cuts = [0, m] if s["offsets"] is None else s["offsets"].tolist()
        loss, grad, alive = 0.0, torch.zeros_like(l), 0
        spans = [(a, b) for a, b in zip(cuts[:-1], cuts[1:]) if int(use[a:b].sum())]
        for a, b in spans:
            u = use[a:b].unsqueeze(1)
            n = int(u.sum())
            i = s["idx"][a:b][use[a:b]].flatten().long()
            f = torch.bincount(i[i >= 0], minlength=e).double() * e / (c["top_k"] * n)
            q = p[a:b] * u
            loss = loss + 0.01 / len(spans) * (f * q.sum(0)).sum() / n
            d = 0.01 / len(spans) / n * q * (f - (q * f).sum(1, keepdim=True))
            grad[a:b] = d * (1 - sg[a:b]) if c["scoring"] == "sigmoid" else d
        n = max(1, int(use.sum()))
        loss = loss + c["z"] * (use * lse * lse).sum() / n
        return {"loss": torch.as_tensor(loss, dtype=torch.float64), "counts": None, "tokens": None, "grad": grad + (c["z"] * 2 / n * use * lse).unsqueeze(1) * sm}

    def weights(w, i, k):
        q, sc, z = (None if t is None else t if i is None else t[i] for t in w)
        v = torch.empty(q.shape[0], k, dtype=torch.float64, device=q.device)
        v[:, 0::2], v[:, 1::2] = (q % 16).double(), (q // 16).double()
        at = torch.arange(k, device=q.device) // c["group"]
        if c["fmt"] == "e2m1":
            sign, size = 1 - 2 * (v >= 8).double(), v % 8
            v = sign * torch.where(size < 2, size / 2, 2.0 ** (torch.floor(size / 2) - 1) * (1 + size % 2 / 2))
            return v * 2.0 ** (sc.double()[:, at] - 127)
        return (v - (8 if z is None else z.double()[:, at])) * sc.double()[:, at]

    x = s["x"].double()
    if c["kind"] == "w4":
        return x @ weights(s["w"], None, c["k"]).t()
    out = torch.zeros_like(x)
    for i in range(c["e"]):
        t, j = (s["idx"] == i).nonzero(as_tuple=True)
        if t.numel():
            up = x[t] @ weights(s["w1"], i, c["k"]).t()
            h = torch.nn.functional.silu(up[:, :c["n"] // 2]) * up[:, c["n"] // 2:]
            out.index_add_(0, t, s["probs"][t, j].double().unsqueeze(1) * (h @ weights(s["w2"], i, c["n"] // 2).t()))
    return out
