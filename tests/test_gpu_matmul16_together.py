"""The products of 16-bit operands, the dense layer and the loss as a program uses them: in one training step behind the gate, recorded as HIP graphs, on other streams and two at
a time, through the native and the general entry path, in the operator library, with long sums, tensors past 2^31 bytes and a vocabulary of several pieces."""
import pytest
import torch

import catccos_amd as cc
import catccos_amd.torch_library  # noqa: F401
import test_gpu_grouped_matmul as grouped
import test_gpu_linear_cross_entropy as loss_test
from bounds16 import check, rounded, sum_error
from catccos_amd import ops

pytestmark = pytest.mark.gpu
OPS = torch.ops.catccos


def same(a, b):
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8))


def flat(r):
    return [t for t in (r if isinstance(r, tuple) else (r,)) if t is not None]


def calls(seed=1):
    """(function, arguments by position): every operator, at sizes that reach each of its kernels, whole rows and rows that have to be padded."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda dtype, *shape: torch.randn(*shape, device="cuda", generator=g).to(dtype)   # noqa: E731
    out = []
    for dtype in (torch.bfloat16, torch.float16):
        for sizes, rest, k, n in (([1, 0], 0, 64, 48), ([70, 0, 45], 9, 136, 200), ([40, 3], 2, 77, 33), ([600, 700, 100], 50, 256, 1032)):
            gs = torch.tensor(sizes, dtype=torch.int32, device="cuda")
            for trans_b in (0, 1):
                x, w = new(dtype, sum(sizes) + rest, k), new(dtype, len(sizes), *((n, k) if trans_b else (k, n)))
                out += [(cc.grouped_matmul, (x, w, gs, trans_b)), (cc.grouped_matmul_backward, (new(dtype, sum(sizes) + rest, n), x, w, gs, trans_b, True, True)),
                        (cc.grouped_matmul_backward, (new(dtype, sum(sizes) + rest, n), x, w, gs, trans_b, False, True))]
        for m, k, n, act in ((1, 1024, 520, "silu"), (40, 77, 131, "gelu"), (256, 4096, 512, "none"), (2100, 520, 2056, "gelu_tanh")):
            for trans_b in (0, 1):
                x, w, b, r = new(dtype, m, k), new(dtype, *((n, k) if trans_b else (k, n))) * k ** -0.5, new(dtype, n), new(dtype, m, n)
                out += [(cc.matmul_bias_act, (x, w, b, r, act, trans_b, True)), (cc.matmul_bias_act, (x, w, None, None, "none", trans_b, False)),
                        (cc.matmul_bias_act_backward, (r, x, w, new(dtype, m, n), act, trans_b, True, True, True)),
                        (cc.matmul_bias_act_backward, (r, x, w, None, "none", trans_b, True, False, True))]
        for t, h, v in ((1, 64, 200), (130, 136, 520), (300, 77, 333), (3000, 128, 5000)):
            x, w = new(dtype, t, h), new(dtype, v, h) * h ** -0.5
            tg = torch.randint(-v // 3, v, (t,), device="cuda", generator=g)
            _, _, lse, tokens = cc.linear_cross_entropy(x, w, tg)
            one = torch.tensor(0.7, device="cuda")
            out += [(cc.linear_cross_entropy, (x, w, tg, "mean", 1e-3)), (cc.linear_cross_entropy, (x, w, tg.int(), "sum", 0.0)),
                    (cc.linear_cross_entropy_backward, (one, x, w, tg, lse, tokens, "mean", 1e-3, True, True)),
                    (cc.linear_cross_entropy_backward, (one, x, w, tg.int(), lse, tokens, "sum", 0.0, True, False))]
    return out


class Declines:
    def __getattr__(self, name):
        return lambda *a: NotImplemented


def test_native_and_general_forms_give_the_same(monkeypatch):
    todo = calls()
    native = [flat(f(*a)) for f, a in todo]
    took, module = [], ops._direct

    class Counts:
        def __getattr__(self, name):
            def f(*a):
                r = getattr(module, name)(*a)
                took.append(r is not NotImplemented)
                return r
            return f
    monkeypatch.setattr(ops, "_direct", Counts())
    for f, a in todo:
        del took[:]
        f(*a)
        assert took == [True], f.__name__
    monkeypatch.setattr(ops, "_direct", Declines())
    for (f, a), got in zip(todo, native):
        want = flat(f(*a))
        assert len(got) == len(want) and all(same(x, y) and not x.requires_grad for x, y in zip(got, want)), f.__name__


def test_what_is_refused_by_one_is_refused_by_both(monkeypatch):
    def outcome(f, a):
        try:
            return [tuple(t.shape) for t in flat(f(*a))]
        except Exception as e:
            return type(e), str(e)
    bad = []
    for f, a in calls()[::9]:
        for i, v in enumerate(a):
            others = (v.cpu(), v.to(torch.float64), v[None], None) if isinstance(v, torch.Tensor) else ("nonsense", None)
            bad += [(f, a[:i] + (o,) + a[i + 1:]) for o in others]
    got = [outcome(*c) for c in bad]
    monkeypatch.setattr(ops, "_direct", Declines())
    for c, g in zip(bad, got):
        assert outcome(*c) == g, c[0].__name__


def test_the_operator_library_gives_the_same():
    assert OPS.finalize() == 0
    with pytest.raises(RuntimeError, match="not initialized"):
        OPS.matmul_bias_act(torch.zeros(4, 16, device="cuda").half(), torch.zeros(16, 8, device="cuda").half(), None, None, "none", 0, False)
    assert OPS.init(0, 1, 1 << 20, "tcp://127.0.0.1:8666") == 0
    for f, a in calls():
        got, want = getattr(OPS, f.__name__)(*a), f(*a)
        got, want = (r if isinstance(r, tuple) else (r,) for r in (got, want))
        for i, (x, y) in enumerate(zip(got, want)):
            assert x.numel() == 0 if y is None else same(x, y), (f.__name__, i)
        if f is cc.matmul_bias_act and not a[-1]:
            assert got[1].numel() == 0
        if "backward" in f.__name__:
            continue
        grads = []
        for lib in (OPS, cc):
            leaves = [v.clone().requires_grad_() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for v in a]
            r = getattr(lib, f.__name__)(*leaves)
            r = r[0] if isinstance(r, tuple) else r
            r.backward(torch.ones_like(r) if r.dim() == 0 else torch.linspace(-1, 1, r.numel(), device="cuda").to(r.dtype).view(r.shape))
            grads.append([v.grad for v in leaves if isinstance(v, torch.Tensor) and v.is_floating_point()])
        assert all(same(x, y) for x, y in zip(*grads)), f.__name__
    x = torch.zeros(4, 16, device="cuda").half()
    for bad in (lambda: OPS.matmul_bias_act(x, torch.zeros(8, 16, device="cuda").half(), None, None, "none", 0, False),
                lambda: OPS.matmul_bias_act(x, torch.zeros(16, 8).half(), None, None, "none", 0, False),
                lambda: OPS.matmul_bias_act(x, torch.zeros(16, 8, device="cuda").half(), x[0], None, "none", 0, False),
                lambda: OPS.matmul_bias_act(x, torch.zeros(16, 8, device="cuda").half(), None, x, "none", 0, False),
                lambda: OPS.grouped_matmul(x, torch.zeros(2, 16, 8, device="cuda").half(), torch.zeros(3, dtype=torch.int32, device="cuda"), 0),
                lambda: OPS.linear_cross_entropy(x, x, torch.zeros(4, device="cuda"), "mean", 0.0),
                lambda: OPS.matmul_bias_act_backward(x, x, torch.zeros(16, 16, device="cuda").half(), None, "silu", 0, True, True, True)):
        with pytest.raises(RuntimeError):
            bad()
    assert OPS.finalize() == 0


def test_on_another_stream_and_in_a_graph():
    todo = calls()
    want = [flat(f(*a)) for f, a in todo]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [flat(f(*a)) for f, a in todo]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [flat(f(*a)) for f, a in todo]
    for _ in range(4):
        for h in held:
            for t in h:
                t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for (f, _), w, o, h in zip(todo, want, other, held):
            for x, y, z in zip(w, o, h):
                assert same(x, y) and same(x, z), f.__name__


def test_two_streams_at_a_time():
    """The same calls on different values, issued in turn on two streams without a wait between them: neither's workspaces or results reach the other's."""
    todo = [calls(1), calls(2)]
    want = [[flat(f(*a)) for f, a in t] for t in todo]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(2):
        got = [[], []]
        for one, two in zip(*todo):
            for i, (f, a) in enumerate((one, two)):
                with torch.cuda.stream(streams[i]):
                    got[i].append(flat(f(*a)))
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            assert all(same(x, y) for p, q in zip(w, g) for x, y in zip(p, q))


def test_two_graphs_replayed_in_turn():
    """Two recordings that share one memory pool, replayed in turn with eager work between them."""
    todo = calls()[::5]
    want = [flat(f(*a)) for f, a in todo]
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        first = [flat(f(*a)) for f, a in todo]
    with torch.cuda.graph(two, pool=one.pool()):
        second = [flat(f(*a)) for f, a in todo]
    for i in range(4):
        for graph, held in ((one, first), (two, second)):
            graph.replay()
            eager = flat(todo[i][0](*todo[i][1]))
            torch.cuda.synchronize()
            assert all(same(x, y) for p, q in zip(want, held) for x, y in zip(p, q)) and all(same(x, y) for x, y in zip(eager, want[i]))


def test_a_recorded_training_step_follows_new_values():
    """Forward and backward of a layer, the experts and the loss in one graph: every replay equals the eager step on the values that lie there then."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    new = lambda *shape: torch.randn(*shape, device="cuda", generator=gen).bfloat16()   # noqa: E731
    x, w1, b1, we, wv = new(300, 128), new(256, 128) * 0.09, new(256), new(4, 256, 128) * 0.06, new(1000, 128) * 0.09
    sizes, tg, one = torch.tensor([100, 0, 150, 50], dtype=torch.int32, device="cuda"), torch.randint(-100, 1000, (300,), device="cuda", generator=gen), torch.ones((), device="cuda")

    def step():
        y, pre = cc.matmul_bias_act(x, w1, b1, None, "gelu", 1, True)
        z = cc.grouped_matmul(y, we, sizes)
        loss, _, lse, tokens = cc.linear_cross_entropy(z, wv, tg)
        gz, gv = cc.linear_cross_entropy_backward(one, z, wv, tg, lse, tokens)
        gy, ge = cc.grouped_matmul_backward(gz, y, we, sizes)
        return (loss, gv, ge) + cc.matmul_bias_act_backward(gy, x, w1, pre, "gelu", 1)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        x.copy_(new(300, 128))
        sizes.copy_(torch.tensor([[100, 0, 150, 50], [0, 0, 0, 0], [300, 0, 0, 0], [10, 20, 30, 240]][i], dtype=torch.int32))
        tg.copy_(torch.randint(-100 if i < 3 else -100000, 1000, (300,), device="cuda", generator=gen))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(held, step())), i


def test_a_recorded_autograd_step():
    """The same through autograd, of leaves that no eager graph holds."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    new = lambda *shape: torch.randn(*shape, device="cuda", generator=gen).bfloat16()   # noqa: E731
    values = [new(300, 128), new(4, 128, 128) * 0.09, new(1000, 128) * 0.09]
    sizes, tg = torch.tensor([100, 0, 150, 50], dtype=torch.int32, device="cuda"), torch.randint(-100, 1000, (300,), device="cuda", generator=gen)

    def step():
        x, we, wv = (v.detach().requires_grad_() for v in values)
        loss = cc.linear_cross_entropy(cc.matmul_bias_act(cc.grouped_matmul(x, we, sizes), we[1], None, x, "silu"), wv, tg, z_coef=1e-4)[0]
        return (loss.detach(),) + torch.autograd.grad(loss, (x, we, wv))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        for v in values:
            v.copy_(new(*v.shape) * 0.1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(held, step()))


@pytest.mark.parametrize("lib", ["python", "torch.ops"])
def test_a_recorded_backward_of_leaves_that_an_eager_graph_holds_is_refused(lib):
    """The check itself, outside any capture: where the node for a leaf was made on the default stream it says so, else not."""
    x, w = torch.randn(8, 64, device="cuda").bfloat16(), torch.randn(64, 32, device="cuda").bfloat16()
    seen = []

    class Look(torch.autograd.Function):
        @staticmethod
        def forward(ctx, v):
            return v.clone()

        @staticmethod
        def backward(ctx, g):
            seen.append(ops._direct.accumulates_on_default_stream())
            return g

    leaf = x.clone().requires_grad_()
    Look.apply(leaf).sum().backward()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fresh = x.clone().requires_grad_()
        Look.apply(fresh).sum().backward()
        Look.apply(fresh * 2).sum().backward()
    torch.cuda.current_stream().wait_stream(side)
    assert seen == [True, False, False]
    assert ops._direct.accumulates_on_default_stream() is False   # (no node runs)
    # what the operators make of it, the capture being told by the test
    leaf = w.clone().requires_grad_()
    if lib == "python":
        y = cc.matmul_bias_act(x, leaf)
        with pytest.MonkeyPatch.context() as patch:
            patch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
            with pytest.raises(RuntimeError, match="eager graph"):
                y.sum().backward()
            with torch.cuda.stream(side):
                ours = w.clone().requires_grad_()
                cc.matmul_bias_act(x, ours).sum().backward()
        torch.cuda.synchronize()
        assert ours.grad is not None
    else:
        assert OPS.init(0, 1, 1 << 20, "tcp://127.0.0.1:8666") == 0
        OPS.matmul_bias_act(x, leaf, None, None, "none", 0, False)[0].sum().backward()
        assert OPS.finalize() == 0 and leaf.grad is not None


def test_a_training_step_of_experts():
    """Gate, routing, the experts' two products, the layer behind them and the loss, with the balance loss: every stage's result and gradient is that of its formula at the
    values that reached it."""
    gen = torch.Generator().manual_seed(7)
    t, h, e, f, v, top_k = 200, 64, 8, 96, 500, 2
    x = torch.randn(t, h, generator=gen).bfloat16()
    gate = (torch.randn(e, h, generator=gen) * h ** -0.5).bfloat16()
    w1, w2 = ((torch.randn(*s, generator=gen) * s[1] ** -0.5).bfloat16() for s in ((e, h, f), (e, f, h)))
    wo, bo, wv = (torch.randn(h, h, generator=gen) * h ** -0.5).bfloat16(), torch.randn(h, generator=gen).bfloat16(), (torch.randn(v, h, generator=gen) * h ** -0.5).bfloat16()
    tg = torch.randint(-50, v, (t,), generator=gen)
    leaves = [p.cuda().requires_grad_() for p in (x, gate, w1, w2, wo, bo, wv)]
    xc, gc, w1c, w2c, woc, boc, wvc = leaves

    logits = cc.matmul_bias_act(xc, gc, trans_b=1)
    probs, idx = cc.moe_router(logits, top_k)
    balance, counts, _ = cc.moe_balance_loss(logits, idx, 0.01, 1e-4)
    order, place, sizes = cc.moe_init_routing(idx, e)
    assert torch.equal(sizes, counts)
    rows = xc[order.long() // top_k]
    a = cc.grouped_matmul(rows, w1c, sizes)
    b = torch.nn.functional.silu(a)
    c = cc.grouped_matmul(b, w2c, sizes)
    mixed = (c[place.long()].view(t, top_k, h) * probs[..., None]).sum(1).bfloat16()
    y = cc.matmul_bias_act(mixed, woc, boc, xc, "gelu")
    loss, nll, lse, tokens = cc.linear_cross_entropy(y, wvc, tg.cuda(), z_coef=1e-4)
    kept = [logits, rows, a, b, c, mixed, y]
    for s in kept:
        s.retain_grad()
    (loss + balance).backward()

    on_host = lambda s: s.detach().cpu()   # noqa: E731
    ns = sizes.tolist()
    loss_test._verify(on_host(y), wv, tg, tuple(on_host(s) for s in (loss, nll, lse, tokens)), None, 1e-4)
    # y.grad comes from the loss alone
    loss_test._verify(on_host(y), wv, tg, tuple(on_host(s) for s in (loss, nll, lse, tokens)), (on_host(y.grad), on_host(wvc.grad)), 1e-4)
    grouped._verify(on_host(a), on_host(rows), w1, ns, 0, on_host(a.grad), (on_host(rows.grad), on_host(w1c.grad)))
    grouped._verify(on_host(c), on_host(b), w2, ns, 0, on_host(c.grad), (on_host(b.grad), on_host(w2c.grad)))
    # the layer: its float64 form at the same operands, its slope at the rounded sum
    z = on_host(mixed).double() @ wo.double() + bo.double()
    ez = sum_error(on_host(mixed).double(), wo.double()) + 2.0 ** -23 * z.abs()
    want = torch.nn.functional.gelu(z) + x.double()
    check(on_host(y), want, rounded(want, 1.13 * ez + 2.0 ** -19 * (z.abs() + 1) + 2.0 ** -23 * want.abs(), torch.bfloat16), "y")
    ez = rounded(z, ez, torch.bfloat16)
    slope = torch.autograd.functional.vjp(torch.nn.functional.gelu, z, on_host(y.grad).double())[1]
    # |gelu''| < 0.8: the slope where z is off by ez, then the rounding of dz
    ed = rounded(slope, on_host(y.grad).double().abs() * (0.8 * ez + 2.0 ** -18), torch.bfloat16)
    gm = slope @ wo.double().t()
    check(on_host(mixed.grad), gm, rounded(gm, ed @ wo.double().abs().t() + sum_error(slope.abs() + ed, wo.double().t()), torch.bfloat16), "mixed")
    gw = on_host(mixed).double().t() @ slope
    check(on_host(woc.grad), gw, rounded(gw, on_host(mixed).double().abs().t() @ ed + sum_error(on_host(mixed).double().t(), slope.abs() + ed), torch.bfloat16), "wo")
    # the gate's layer: its gradient is its product's
    gl = on_host(logits.grad).double()
    want = gl.t() @ x.double()
    check(on_host(gc.grad), want, rounded(want, sum_error(gl.t(), x.double()), torch.bfloat16), "gate")
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) and bool(p.grad.any()) for p in leaves)


@pytest.mark.parametrize("m,k,n", [(256, 4096, 512), (130, 7000, 136), (1, 16384, 96), (40, 8200, 1000)])
@pytest.mark.parametrize("trans_b", [0, 1])
def test_long_sums(m, k, n, trans_b):
    """Few tiles and a long K, which is split over workgroups: the same bits every time, within the bound of a sum of k terms."""
    gen = torch.Generator().manual_seed(8)
    x, w = torch.randn(m, k, generator=gen).bfloat16(), (torch.randn(*((n, k) if trans_b else (k, n)), generator=gen) * k ** -0.5).bfloat16()
    b = torch.randn(n, generator=gen).bfloat16()
    wk = (w.t() if trans_b else w).double()
    z = x.double() @ wk + b.double()
    got = cc.matmul_bias_act(x.cuda(), w.cuda(), b.cuda(), trans_b=trans_b)
    check(got, z, rounded(z, sum_error(x.double(), wk) + 2.0 ** -23 * z.abs(), torch.bfloat16))
    for _ in range(3):
        assert torch.equal(cc.matmul_bias_act(x.cuda(), w.cuda(), b.cuda(), trans_b=trans_b), got)
    # the weights' gradient of a product with few columns and many rows, likewise
    gx, gw, gb = cc.matmul_bias_act_backward(torch.randn(k, n, generator=gen).bfloat16().cuda(), torch.randn(k, m, generator=gen).bfloat16().cuda(),
                                             torch.zeros((n, m) if trans_b else (m, n)).bfloat16().cuda(), trans_b=trans_b)
    gen = torch.Generator().manual_seed(8)
    for s in ((m, k), (n, k) if trans_b else (k, n), (n,)):
        torch.randn(*s, generator=gen)
    g, x = torch.randn(k, n, generator=gen).bfloat16().double(), torch.randn(k, m, generator=gen).bfloat16().double()
    want, bound = x.t() @ g, sum_error(x.t(), g)
    want, bound = (want.t(), bound.t()) if trans_b else (want, bound)
    check(gw, want, rounded(want, bound, torch.bfloat16))
    assert not gx.any()


@pytest.fixture
def big_tiles():
    cc.set_option("matmul16_kernel", 1)
    yield
    cc.set_option("matmul16_kernel", -1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("trans_b", [0, 1])
@pytest.mark.parametrize("sizes,rest,k,n", [([300, 1, 0, 129, 600], 7, 4096, 520), ([40], 0, 9999, 33), ([2000, 0, 900, 1800], 5, 4424, 4400)])
def test_tiles_of_256_and_a_long_k_in_groups(big_tiles, sizes, rest, k, n, trans_b, dtype):
    """K is worked on in parts where the last round of tiles leaves workgroups idle: behind whole rounds (some 340 tiles) and alone."""
    x, w, g, gs = (v.cuda() for v in grouped._case(sizes, rest, k, n, trans_b, dtype))
    out = cc.grouped_matmul(x, w, gs, trans_b)
    grads = cc.grouped_matmul_backward(g, x, w, gs, trans_b)
    assert same(out, cc.grouped_matmul(x, w, gs, trans_b))
    for (a, b), i in zip(grouped._ranges(sizes, x.shape[0]), range(len(sizes))):
        m = (w[i].t() if trans_b else w[i]).double()
        want = x[a:b].double() @ m
        check(out[a:b], want, rounded(want, sum_error(x[a:b].double(), m), dtype), "out %d" % i)
        want = g[a:b].double() @ m.t()
        check(grads[0][a:b], want, rounded(want, sum_error(g[a:b].double(), m.t()), dtype), "grad_x %d" % i)
    assert not out[sum(sizes):].any() and not grads[0][sum(sizes):].any()


@pytest.mark.parametrize("m,k,n,act", [(700, 4200, 520, "gelu"), (4400, 4096, 4100, "silu"), (1, 20000, 8, "none"), (257, 65600, 256, "relu")])
@pytest.mark.parametrize("trans_b", [0, 1])
def test_tiles_of_256_and_a_long_k_in_a_layer(big_tiles, m, k, n, act, trans_b):
    gen = torch.Generator(device="cuda").manual_seed(11)
    new = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)   # noqa: E731
    x, w, b, r = new(m, k).bfloat16(), (new(*((n, k) if trans_b else (k, n))) * k ** -0.5).bfloat16(), new(n).bfloat16(), new(m, n).bfloat16()
    wk = (w.t() if trans_b else w).double()
    z = x.double() @ wk + b.double()
    ez = sum_error(x.double(), wk) + 2.0 ** -23 * z.abs()
    y = {"gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu, "relu": torch.relu, "none": lambda v: v}[act](z) + r.double()
    out, pre = cc.matmul_bias_act(x, w, b, r, act, trans_b, True)
    check(pre, z, rounded(z, ez, torch.bfloat16), "preact")
    check(out, y, rounded(y, 1.13 * ez + 2.0 ** -19 * (z.abs() + 1) + 2.0 ** -23 * y.abs(), torch.bfloat16), "out")
    assert all(same(a, c) for a, c in zip((out, pre), cc.matmul_bias_act(x, w, b, r, act, trans_b, True)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,h,v", [(66000, 24, 3700), (16000, 264, 9000)])
def test_a_vocabulary_of_several_pieces(t, h, v, dtype):
    """Enough tokens that the gradient of the logits is worked on in several pieces, whose shares of grad_x are added up; the second, of pieces of more than 4096
    columns, sums them in parts."""
    x, w, tg = loss_test._case(t, h, v, dtype, 0.6)
    scale = 1024.0 if dtype == torch.float16 else 1.0
    got = cc.linear_cross_entropy(x.cuda(), w.cuda(), tg.cuda(), reduction="sum", z_coef=1e-4)
    grads = cc.linear_cross_entropy_backward(torch.full((), scale, device="cuda"), x.cuda(), w.cuda(), tg.cuda(), got[2], got[3], reduction="sum", z_coef=1e-4)
    loss_test._verify(x, w, tg, got, grads, 1e-4, "sum", scale)
    again = cc.linear_cross_entropy_backward(torch.full((), scale, device="cuda"), x.cuda(), w.cuda(), tg.cuda(), got[2], got[3], reduction="sum", z_coef=1e-4)
    assert all(same(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("kernel", [0, 1])
def test_logits_of_minus_infinity_count_nothing(kernel):
    """Columns whose logit is -inf for every token, a whole run of 64 of them among others: the loss is that without them; a NaN logit is not lost there."""
    gen = torch.Generator().manual_seed(12)
    x = (torch.rand(70, 40, generator=gen) + 0.1).bfloat16()
    w = (torch.randn(400, 40, generator=gen) * 0.2).bfloat16()
    out = torch.zeros(400, dtype=torch.bool)
    out[64:128] = out[200:210] = out[399] = True
    tg = torch.arange(400)[~out][torch.randint(int((~out).sum()), (70,), generator=gen)]
    w[out, 3] = float("-inf")
    l = x.double() @ w[~out].double().t()
    el = sum_error(x.double(), w[~out].double().t())
    want = torch.logsumexp(l, 1)
    bound = el.amax(1) + loss_test.EXP + 130 * 2.0 ** -24 + 2.0 ** -22 * want.abs()
    cc.set_option("matmul16_kernel", kernel)
    try:
        got = cc.linear_cross_entropy(x.cuda(), w.cuda(), tg.cuda())
        check(got[2], want, bound, "lse")
        x[5, 3] = float("nan")
        lse = cc.linear_cross_entropy(x.cuda(), w.cuda(), tg.cuda())[2]
    finally:
        cc.set_option("matmul16_kernel", -1)
    assert torch.isnan(lse[5]) and int(torch.isnan(lse).sum()) == 1


@pytest.mark.parametrize("trans_b", [0, 1])
def test_tensors_past_32_bits(trans_b):
    """x, out and the weights each beyond 2^31 bytes: what lies behind that is where it belongs."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    new = lambda *shape: torch.randn(*shape, device="cuda", generator=gen).bfloat16()   # noqa: E731
    m, last = 300001, slice(299700, 300001)
    x, w = new(m, 4096), new(*((64, 4096) if trans_b else (4096, 64))) / 64
    wk = (w.t() if trans_b else w).double().cpu()
    out = cc.matmul_bias_act(x, w, trans_b=trans_b)
    xl = x[last].double().cpu()
    want = xl @ wk
    check(out[last], want, rounded(want, sum_error(xl, wk), torch.bfloat16), "x")
    # the weights' gradient where only the last rows have one
    g = torch.zeros(m, 64, device="cuda", dtype=torch.bfloat16)
    g[last] = new(301, 64)
    gw = cc.matmul_bias_act_backward(g, x, w, trans_b=trans_b, x_grad=False, bias_grad=False)[1]
    gl = g[last].double().cpu()
    want, bound = xl.t() @ gl, sum_error(xl.t(), gl)
    check(gw.t() if trans_b else gw, want, rounded(want, bound, torch.bfloat16), "grad_w")
    # its input's gradient writes past 2^31 bytes
    gx = cc.matmul_bias_act_backward(g, x, w, trans_b=trans_b, w_grad=False, bias_grad=False)[0]
    want = gl @ wk.t()
    check(gx[last], want, rounded(want, sum_error(gl, wk.t()), torch.bfloat16), "grad_x")
    assert not gx[:299700].any()
    del x, g, gx, out
    # the last of the experts
    e = 40
    w = new(e, *((4096, 8192) if trans_b else (8192, 4096))) / 90
    x, sizes = new(50, 8192), torch.zeros(e, dtype=torch.int32, device="cuda")
    sizes[3], sizes[e - 1] = 20, 30
    out = cc.grouped_matmul(x, w, sizes, trans_b)
    gw = cc.grouped_matmul_backward(new(50, 4096), x, w, sizes, trans_b, x_grad=False)[1]
    for rows, i in ((slice(0, 20), 3), (slice(20, 50), e - 1)):
        a, b = x[rows].double().cpu(), (w[i].t() if trans_b else w[i]).double().cpu()
        want = a @ b
        check(out[rows], want, rounded(want, sum_error(a, b), torch.bfloat16), "expert %d" % i)
        assert bool(gw[i].any()) and not gw[i - 1].any()


def test_tensors_of_another_device_than_the_current_one_are_refused_or_served():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    x, w = torch.randn(4, 64, device="cuda:1").half(), torch.randn(64, 32, device="cuda:1").half()
    assert torch.cuda.current_device() == 0
    want = x.double() @ w.double()
    check(cc.matmul_bias_act(x, w), want, rounded(want, sum_error(x.double(), w.double()), torch.float16))
    with pytest.raises(ValueError):
        cc.matmul_bias_act(x, w.to("cuda:0"))
