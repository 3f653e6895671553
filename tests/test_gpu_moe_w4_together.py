"""Router, balance loss and 4-bit products together: recorded as HIP graphs, on other streams, through the native and the general entry path, and in the example
that trains a gate and decodes with it."""
import pytest
import torch

import catccos_amd as cc
from catccos_amd import ops, run_moe_w4

pytestmark = pytest.mark.gpu


def same(a, b):
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8))


def flat(r):
    return r if isinstance(r, tuple) else (r,)


def calls():
    g = torch.Generator(device="cuda").manual_seed(1)
    out = []
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for t, e, k in ((1, 16, 6), (37, 64, 8), (700, 100, 3)):
            logits = torch.randn(t, e, device="cuda", generator=g).to(dtype)
            mask = torch.rand(t, device="cuda", generator=g) < 0.8
            bias = torch.randn(e, device="cuda", generator=g) * 0.1
            offsets = torch.tensor([0, t // 3, t // 3, t], dtype=torch.int32, device="cuda")
            for scoring in ("softmax", "sigmoid"):
                probs, idx = cc.moe_router(logits, k, scoring, True, 2.5, bias, mask)
                grad = torch.randn(t, k, device="cuda", generator=g)
                one = torch.tensor(0.7, device="cuda")
                out += [(cc.moe_router, (logits, k), {}), (cc.moe_router, (logits, k, scoring, True, 2.5, bias, mask), {}),
                        (cc.moe_router, (logits, k), {"scoring": scoring, "renormalize": False, "token_mask": mask}),
                        (cc.moe_router_backward, (grad, logits, idx, scoring, False, 1.5), {})]
                for off in (None, offsets):
                    kw = {"scoring": scoring, "token_mask": mask, "seq_offsets": off}
                    _, counts, counted = cc.moe_balance_loss(logits, idx, 0.1, 1e-3, **kw)
                    out += [(cc.moe_balance_loss, (logits, idx, 0.1, 1e-3), kw), (cc.moe_balance_loss_backward, (one, logits, counts, counted, k, 0.1, 1e-3), kw)]
    for dtype in (torch.bfloat16, torch.float16):
        for fmt, group, zeros in (("int4", 128, True), ("int4", 32, False), ("e2m1", 32, False)):
            def w(*shape):
                codes = torch.randint(0, 256, shape[:-1] + (shape[-1] // 2,), device="cuda", generator=g, dtype=torch.uint8)
                if fmt == "e2m1":
                    return codes, torch.randint(118, 124, shape[:-1] + (cc.scale_cols(shape[-1]),), device="cuda", generator=g, dtype=torch.uint8), None
                s = (torch.rand(shape[:-1] + ((shape[-1] + group - 1) // group,), device="cuda", generator=g) * 0.02).to(dtype)
                return codes, s, torch.randint(0, 16, s.shape, device="cuda", generator=g, dtype=torch.uint8) if zeros else None
            for m in (1, 8, 40):
                x = torch.randn(m, 256, device="cuda", generator=g).to(dtype)
                probs, idx = cc.moe_router(torch.randn(m, 6, device="cuda", generator=g), 2)
                out += [(cc.w4a16_matmul, (x,) + w(96, 256), {"fmt": fmt, "group_size": group}),
                        (cc.moe_ffn_w4a16, (x, idx, probs) + w(6, 128, 256) + w(6, 256, 64), {"fmt": fmt, "group_size": group})]
    return out


class Declines:
    def __getattr__(self, name):
        return lambda *a: NotImplemented


def test_native_and_general_forms_give_the_same(monkeypatch):
    todo = calls()
    native = [flat(f(*a, **kw)) for f, a, kw in todo]
    took = []
    module = ops._direct

    class Counts:
        def __getattr__(self, name):
            def f(*a):
                r = getattr(module, name)(*a)
                took.append(r is not NotImplemented)
                return r
            return f
    monkeypatch.setattr(ops, "_direct", Counts())
    for f, a, kw in todo:
        del took[:]
        f(*a, **kw)
        assert took == [True], f.__name__
    monkeypatch.setattr(ops, "_direct", Declines())
    for (f, a, kw), got in zip(todo, native):
        want = flat(f(*a, **kw))
        assert len(got) == len(want)
        for x, y in zip(got, want):
            assert same(x, y) and not x.requires_grad, f.__name__


def test_what_was_refused_stays_refused(monkeypatch):
    def outcome(f, a, kw):
        try:
            return [tuple(t.shape) for t in flat(f(*a, **kw))]
        except Exception as e:
            return type(e), str(e)
    bad = []
    for f, a, kw in calls()[::7]:
        for i, v in enumerate(a):
            others = (v.cpu(), v.to(torch.float64), v[None], None) if isinstance(v, torch.Tensor) else ("nonsense", None)
            bad += [(f, a[:i] + (o,) + a[i + 1:], kw) for o in others]
        bad += [(f, a, {**kw, name: "nonsense"}) for name in ("scoring", "fmt") if name in kw]
    got = [outcome(*c) for c in bad]
    monkeypatch.setattr(ops, "_direct", Declines())
    for c, g in zip(bad, got):
        assert outcome(*c) == g, c[0].__name__


def test_on_another_stream_and_in_a_graph():
    todo = calls()
    want = [flat(f(*a, **kw)) for f, a, kw in todo]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [flat(f(*a, **kw)) for f, a, kw in todo]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [flat(f(*a, **kw)) for f, a, kw in todo]
    for _ in range(4):
        for h in held:
            for t in h:
                t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for (f, _, _), w, o, h in zip(todo, want, other, held):
            for x, y, z in zip(w, o, h):
                assert same(x, y) and same(x, z), f.__name__


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_a_recorded_training_step_follows_new_logits(scoring):
    """Forward and backward of router and losses in one graph: every replay equals the eager step on the values that lie there then."""
    torch.manual_seed(0)
    logits = torch.randn(300, 32, device="cuda")
    probs_grad = torch.randn(300, 4, device="cuda")
    one = torch.ones((), device="cuda")

    def step():
        probs, idx = cc.moe_router(logits, 4, scoring)
        loss, counts, counted = cc.moe_balance_loss(logits, idx, 0.1, 1e-3, scoring)
        grad = cc.moe_router_backward(probs_grad, logits, idx, scoring) + cc.moe_balance_loss_backward(one, logits, counts, counted, 4, 0.1, 1e-3, scoring)
        return probs, idx, loss, counts, grad

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(4):
        logits.copy_(torch.randn(300, 32, device="cuda") * 2)
        for t in held:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for h, w in zip(held, step()):
            assert same(h, w)
    # and autograd's gradient is the sum of the two
    leaf = logits.clone().requires_grad_()
    probs, idx = cc.moe_router(leaf, 4, scoring)
    loss, _, _ = cc.moe_balance_loss(leaf, idx, 0.1, 1e-3, scoring)
    (loss + (probs * probs_grad).sum()).backward()
    assert torch.allclose(leaf.grad, step()[4], rtol=1e-6, atol=1e-8)


@pytest.mark.parametrize("options", [[], ["--fmt", "e2m1", "--scoring", "sigmoid", "--batch", "3"], ["--half", "--group", "32", "--batch", "20"]])
def test_example(options):
    assert run_moe_w4.main(["--tokens", "1024", "--steps", "30", "--k", "512", "--n", "256", "--vocab", "1000", "--replays", "5"] + options) == 0
