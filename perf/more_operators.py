"""The products in 16 bits that training and serving ask for next to the quantised ones, and the loss at their end.

Three operators, each called as a user's program calls it:

    gmm     tokens sorted by expert times each expert's weights, groups of any sizes; in training the tokens' and the weights' gradient too
    linear  a dense product whose epilogue adds the bias, applies the activation and adds the residual; or its backward pass
    ce      softmax cross entropy of hidden states against an output projection, without the logits; in training both gradients

`run` computes them from the formulas with elementary torch operations in 32 bits, or, where `own` is true, calls the package.
Sizes of layers are those of this repository's configurations and shape lists, and in draw() others of the same kind."""
import math

import torch

own = False


def listed():
    return [
        # the routes of one token through 64 small experts, a decode step: eight experts' weights are read for a row each
        {"name": "gmm-one", "kind": "gmm", "t": 8, "e": 64, "k": 2048, "n": 1024, "trans": 1, "half": False, "skew": 0.0, "tail": 0.0, "backward": False},
        # a prompt's routes through an up projection, weights [K, N]
        {"name": "gmm-prompt", "kind": "gmm", "t": 4096, "e": 16, "k": 7168, "n": 4096, "trans": 0, "half": False, "skew": 0.5, "tail": 0.0, "backward": False},
        # a training step through the largest expert layer there is, with both gradients
        {"name": "gmm-train", "kind": "gmm", "t": 16384, "e": 32, "k": 7168, "n": 4096, "trans": 1, "half": False, "skew": 0.3, "tail": 0.0, "backward": True},
        # very uneven groups, some empty, rows behind the last of them, sizes that fill no tile, in halves
        {"name": "gmm-ragged", "kind": "gmm", "t": 5003, "e": 20, "k": 1984, "n": 1000, "trans": 1, "half": True, "skew": 1.6, "tail": 0.1, "backward": True},
        # one token of a decode step
        {"name": "linear-one", "kind": "linear", "m": 1, "k": 7168, "n": 4096, "trans": 1, "half": False, "act": "silu", "bias": True, "residual": True,
         "preact": False, "backward": False},
        # a short prompt
        {"name": "linear-512", "kind": "linear", "m": 512, "k": 2048, "n": 7168, "trans": 1, "half": False, "act": "gelu_tanh", "bias": True, "residual": False,
         "preact": False, "backward": False},
        # the largest layer there is, as training calls it: what the activation was applied to is kept
        {"name": "linear-16384", "kind": "linear", "m": 16384, "k": 7168, "n": 4096, "trans": 0, "half": False, "act": "gelu", "bias": True, "residual": True,
         "preact": True, "backward": False},
        # a layer's backward pass: gradients of the input, the weights and the bias
        {"name": "linear-back", "kind": "linear", "m": 8192, "k": 2048, "n": 7168, "trans": 1, "half": False, "act": "gelu_tanh", "bias": True, "residual": False,
         "preact": True, "backward": True},
        # the same of a layer whose rows start on no boundary, in halves
        {"name": "linear-odd-back", "kind": "linear", "m": 333, "k": 1111, "n": 777, "trans": 1, "half": True, "act": "silu", "bias": True, "residual": False,
         "preact": True, "backward": True},
        # the likelihood of a short text
        {"name": "ce-text", "kind": "ce", "t": 256, "h": 2048, "v": 8192, "half": False, "pad": 0.0, "z": 0.0, "backward": False},
        # the head of a training step, loss and both gradients
        {"name": "ce-train", "kind": "ce", "t": 8192, "h": 4096, "v": 32768, "half": False, "pad": 0.0, "z": 0.0, "backward": True},
        # a ragged batch most of whose tokens are prompt, which do not count, with the z loss, in halves
        {"name": "ce-masked", "kind": "ce", "t": 4999, "h": 1984, "v": 20011, "half": True, "pad": 0.6, "z": 1e-4, "backward": True},
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _dim(rng, lo, hi):
    """A layer's size: some a power of two, some a multiple of 128 or 8, some anything."""
    v = _log(rng, lo, hi)
    u = rng.choice([0, 128, 128, 8, 8, 1])
    return max(lo, 1 << v.bit_length() - 1 if u == 0 else v // u * u)


def draw(rng):
    while True:
        kind = rng.choice(["gmm", "linear", "ce"])
        c = {"kind": kind, "half": rng.random() < 0.3}
        if kind == "gmm":
            c.update(t=_log(rng, 1, 16384), e=rng.choice([2, 4, 8, 16, 20, 32, 60, 64, 128]), k=_dim(rng, 256, 8192), n=_dim(rng, 256, 8192), trans=rng.choice([0, 1]),
                     skew=rng.choice([0.0, 0.3, 0.5, 1.0, 1.6]), tail=rng.choice([0.0, 0.0, 0.1]), backward=rng.random() < 0.5)
            if c["e"] * c["k"] * c["n"] <= 32 * 7168 * 4096 and c["t"] * c["k"] * c["n"] <= 16384 * 7168 * 4096:
                return c
        elif kind == "linear":
            c.update(m=_log(rng, 1, 16384), k=_dim(rng, 256, 8192), n=_dim(rng, 256, 8192), trans=rng.choice([0, 1]),
                     act=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]), bias=rng.random() < 0.7, residual=rng.random() < 0.5,
                     preact=rng.random() < 0.5, backward=rng.random() < 0.4)
            if c["backward"]:
                c.update(residual=False, preact=True)
            if c["m"] * c["k"] * c["n"] <= 16384 * 7168 * 4096 / (2 if c["backward"] else 1):
                return c
        else:
            c.update(t=_log(rng, 1, 16384), h=_dim(rng, 256, 8192), v=_dim(rng, 1024, 131072), pad=rng.choice([0.0, 0.0, 0.3, 0.6]), z=rng.choice([0.0, 1e-4]),
                     backward=rng.random() < 0.6)
            if c["t"] * c["h"] * c["v"] <= 8192 * 4096 * 32768 and c["h"] * c["v"] <= 8192 * 65536:
                return c


def _activations(gen, m, k, dtype):
    """Activations as a normalisation leaves them: unit variance, a few channels an order of magnitude larger."""
    gain = torch.exp(0.5 * torch.randn(k, device="cuda", generator=gen))
    return (torch.randn(m, k, device="cuda", generator=gen) * gain).to(dtype)


def _weights(gen, *shape, fan, dtype):
    return (torch.randn(*shape, device="cuda", generator=gen) * fan ** -0.5).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    c = dict(case)
    dtype = torch.float16 if c["half"] else torch.bfloat16
    s = {"case": c}
    if c["kind"] == "gmm":
        t, e, k, n = c["t"], c["e"], c["k"], c["n"]
        share = torch.exp(c["skew"] * torch.randn(e, device="cuda", generator=gen))
        rows = t - int(t * c["tail"])
        to = torch.multinomial(share, rows, replacement=True, generator=gen)
        s["group_sizes"] = torch.bincount(to, minlength=e).to(torch.int32)
        s["sizes"] = s["group_sizes"].tolist()           # the plain form's plan: its slices have to be known to the host
        s["x"] = _activations(gen, t, k, dtype)
        s["w"] = _weights(gen, *((e, n, k) if c["trans"] else (e, k, n)), fan=k, dtype=dtype)
        if c["backward"]:
            s["grad"] = torch.randn(t, n, device="cuda", generator=gen).to(dtype)
    elif c["kind"] == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        s["x"] = _activations(gen, m, k, dtype)
        s["w"] = _weights(gen, *((n, k) if c["trans"] else (k, n)), fan=k, dtype=dtype)
        s["bias"] = _weights(gen, n, fan=4, dtype=dtype) if c["bias"] else None
        s["residual"] = torch.randn(m, n, device="cuda", generator=gen).to(dtype) if c["residual"] else None
        if c["backward"]:
            s["grad"] = torch.randn(m, n, device="cuda", generator=gen).to(dtype)
            s["pre"] = (1.3 * torch.randn(m, n, device="cuda", generator=gen)).to(dtype)     # as the forward pass kept it
    else:
        t, h, v = c["t"], c["h"], c["v"]
        s["w"] = _weights(gen, v, h, fan=h, dtype=dtype)
        s["targets"] = torch.randint(v, (t,), device="cuda", generator=gen)
        # hidden states of a model that has learnt something: a token's logit lies 0 to 12 above the others
        sure = 12 * torch.rand(t, 1, device="cuda", generator=gen)
        s["x"] = (torch.randn(t, h, device="cuda", generator=gen) + sure * s["w"][s["targets"]].float()).to(dtype)
        if c["pad"]:
            s["targets"] = torch.where(torch.rand(t, device="cuda", generator=gen) < c["pad"], -100, s["targets"])
        s["grad"] = torch.full((), 65536.0 if c["half"] else 1.0, device="cuda")   # training in halves scales its loss
    return s


def _plain_gmm(s, c):
    x, sizes, w = s["x"].float(), s["sizes"], s["w"]
    left = c["t"] - sum(sizes)
    xs = x.split(sizes + [left])
    ws = [(w[i].float().t() if c["trans"] else w[i].float()) if r else None for i, r in enumerate(sizes)]     # [K, N] of the experts that have rows
    out = {"out": torch.cat([a @ b for a, b in zip(xs, ws) if b is not None] + [x.new_zeros(left, c["n"])]).to(s["x"].dtype)}
    if c["backward"]:
        gs = s["grad"].float().split(sizes + [left])
        out["grad_x"] = torch.cat([g @ b.t() for g, b in zip(gs, ws) if b is not None] + [x.new_zeros(left, c["k"])]).to(s["x"].dtype)
        pairs = zip(gs[:-1], xs[:-1])
        out["grad_w"] = torch.stack([(g.t() @ a if c["trans"] else a.t() @ g).to(w.dtype) for g, a in pairs])
    return out


def _plain_act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    return z


def _plain_slope(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "silu":
        g = 1 / (1 + torch.exp(-z))
        return g * (1 + z * (1 - g))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if act == "gelu_tanh":
        t = torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * (2 / math.pi) ** 0.5 * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _plain_linear(s, c):
    dtype = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    if c["backward"]:
        d = s["grad"].float() * _plain_slope(s["pre"].float(), c["act"])
        out = {"grad_x": (d @ w if c["trans"] else d @ w.t()).to(dtype), "grad_w": (d.t() @ x if c["trans"] else x.t() @ d).to(dtype)}
        if c["bias"]:
            out["grad_bias"] = d.sum(0).to(dtype)
        return out
    z = x @ (w.t() if c["trans"] else w)
    if c["bias"]:
        z = z + s["bias"].float()
    y = _plain_act(z, c["act"])
    if c["residual"]:
        y = y + s["residual"].float()
    return {"out": y.to(dtype), "preact": z.to(dtype)} if c["preact"] else {"out": y.to(dtype)}


def _plain_ce(s, c):
    x, w = s["x"].float(), s["w"].float()
    there = s["targets"] >= 0
    at = s["targets"].clamp_min(0).unsqueeze(1)
    logits = x @ w.t()
    top = logits.amax(1, keepdim=True)
    ex = torch.exp(logits - top)
    total = ex.sum(1, keepdim=True)
    lse = (torch.log(total) + top).squeeze(1) * there
    nll = (lse - logits.gather(1, at).squeeze(1)) * there
    n = there.sum()
    share = there / n.clamp_min(1)
    loss = (nll.double() * share).sum() + c["z"] * (lse.double() ** 2 * share).sum()
    out = {"loss": loss.float(), "nll": nll, "lse": lse, "tokens": n.to(torch.int32).reshape(1)}
    if c["backward"]:
        d = ex * ((1 + 2 * c["z"] * lse).unsqueeze(1) / total)
        d = d.scatter_add(1, at, torch.full_like(at, -1, dtype=torch.float32)) * (share * s["grad"]).unsqueeze(1)
        out.update(grad_x=(d @ w).to(s["x"].dtype), grad_w=(d.t() @ x).to(s["w"].dtype))
    return out


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"gmm": _plain_gmm, "linear": _plain_linear, "ce": _plain_ce}[c["kind"]](s, c)
    import catccos_amd as cc
    if c["kind"] == "gmm":
        out = {"out": cc.grouped_matmul(s["x"], s["w"], s["group_sizes"], trans_b=c["trans"])}
        if c["backward"]:
            out["grad_x"], out["grad_w"] = cc.grouped_matmul_backward(s["grad"], s["x"], s["w"], s["group_sizes"], trans_b=c["trans"])
        return out
    if c["kind"] == "linear":
        if c["backward"]:
            gx, gw, gb = cc.matmul_bias_act_backward(s["grad"], s["x"], s["w"], s["pre"], activation=c["act"], trans_b=c["trans"], bias_grad=c["bias"])
            return {"grad_x": gx, "grad_w": gw, "grad_bias": gb} if c["bias"] else {"grad_x": gx, "grad_w": gw}
        r = cc.matmul_bias_act(s["x"], s["w"], s["bias"], s["residual"], activation=c["act"], trans_b=c["trans"], return_preact=c["preact"])
        return {"out": r[0], "preact": r[1]} if c["preact"] else {"out": r}
    loss, nll, lse, tokens = cc.linear_cross_entropy(s["x"], s["w"], s["targets"], z_coef=c["z"])
    out = {"loss": loss, "nll": nll, "lse": lse, "tokens": tokens}
    if c["backward"]:
        out["grad_x"], out["grad_w"] = cc.linear_cross_entropy_backward(s["grad"], s["x"], s["w"], s["targets"], lse, tokens, z_coef=c["z"])
    return out


def work(case):
    c = case
    if c["kind"] == "gmm":
        t, k, n = c["t"] * (1 - c["tail"]), c["k"], c["n"]
        read = c["e"] * (1 - (1 - 1 / c["e"]) ** t)              # experts that have rows, about
        if c["backward"]:   # the forward pass, and x, w, the gradient in, two gradients out
            return {"bytes": 2 * (2 * t * (k + n) + read * k * n + t * k + c["e"] * k * n), "flops": 6.0 * t * k * n}
        return {"bytes": 2 * (t * (k + n) + read * k * n), "flops": 2.0 * t * k * n}
    if c["kind"] == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        if c["backward"]:
            return {"bytes": 2 * (2 * m * n + 2 * m * k + 2 * k * n + n * c["bias"]), "flops": 4.0 * m * k * n}
        return {"bytes": 2 * (m * k + k * n + m * n * (1 + c["residual"] + c["preact"]) + n * c["bias"]), "flops": 2.0 * m * k * n}
    t, h, v = c["t"], c["h"], c["v"]
    counted = t * (1 - c["pad"])
    small = 8 * t + 8 * t + 8
    if c["backward"]:   # the loss, and its inputs in and two gradients out
        return {"bytes": 2 * (2 * counted * h + 2 * v * h + t * h + v * h) + 2 * small, "flops": 6.0 * counted * h * v}
    return {"bytes": 2 * (counted * h + v * h) + small, "flops": 2.0 * counted * h * v}


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    x, w = s["x"].double(), s["w"]
    out = {}
    if c["kind"] == "gmm":
        y = x.new_zeros(c["t"], c["n"])
        if c["backward"]:
            g, gx, gw = s["grad"].double(), torch.zeros_like(x), torch.zeros(w.shape, dtype=torch.float64, device=w.device)
        ends = torch.cumsum(s["group_sizes"], 0).tolist()
        for i, end in enumerate(ends):
            rows = slice(ends[i - 1] if i else 0, end)
            if rows.start == end:
                continue
            wi = w[i].double() if not c["trans"] else w[i].double().t()
            y[rows] = torch.mm(x[rows], wi)
            if c["backward"]:
                gx[rows] = torch.mm(g[rows], wi.t())
                d = torch.mm(x[rows].t(), g[rows])
                gw[i] = d.t() if c["trans"] else d
        out["out"] = y
        if c["backward"]:
            out.update(grad_x=gx, grad_w=gw)
        return out
    w = w.double()
    if c["kind"] == "linear":
        f = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
             "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[c["act"]]
        wk = w.t() if c["trans"] else w
        if c["backward"]:
            z = s["pre"].double().requires_grad_()
            d, = torch.autograd.grad(f(z), z, s["grad"].double())
            gw = torch.mm(x.t(), d)
            out = {"grad_x": torch.mm(d, wk.t()), "grad_w": gw.t() if c["trans"] else gw}
            if c["bias"]:
                out["grad_bias"] = d.sum(0)
            return out
        z = torch.mm(x, wk) + (s["bias"].double() if c["bias"] else 0)
        y = f(z) + (s["residual"].double() if c["residual"] else 0)
        return {"out": y, "preact": z} if c["preact"] else {"out": y}
    use = (s["targets"] >= 0).nonzero().squeeze(1)
    n = max(1, use.numel())
    xu, tu = x[use], s["targets"][use]
    logits = torch.mm(xu, w.t())
    lse = torch.logsumexp(logits, 1)
    nll = lse - logits[torch.arange(use.numel(), device=x.device), tu]
    rows = lambda v: torch.zeros((c["t"],) + tuple(v.shape[1:]), dtype=torch.float64, device=x.device).index_copy_(0, use, v)  # noqa: E731
    out = {"loss": nll.sum() / n + c["z"] * (lse * lse).sum() / n, "nll": rows(nll), "lse": rows(lse), "tokens": None}
    if c["backward"]:
        d = torch.softmax(logits, 1) * (1 + 2 * c["z"] * lse).unsqueeze(1)
        d[torch.arange(use.numel(), device=x.device), tu] -= 1
        d *= s["grad"].double() / n
        out.update(grad_x=rows(torch.mm(d, w)), grad_w=torch.mm(d.t(), xu))
    return out
