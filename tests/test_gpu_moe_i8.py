"""A routed layer of int8 experts (K_Q8C stacks through bgl_moe_ffn_dev / bgl_moe_layer_dev) against the plain numpy form,
bit for bit: the integer sums are exact, and codes, SwiGLU and the weighted sums are single fp32 operations in a stated
order (the exponential and the router's sums are doubles, rounded once)."""
import numpy as np
import pytest

import int8_forms as I

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_dev():
    import torch
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    return torch


@pytest.fixture(scope="module")
def ctx(torch_dev):
    import beglin_amd
    c = beglin_amd.Context(0)
    yield c
    c.sync()
    c.close()


class Layer:
    def __init__(self, ctx, seed, E, H, W, Wsh):
        import beglin_amd as B
        rng = np.random.default_rng(seed)
        self.parts = [[I.weights(rng, o, k) for _ in range(E)] for o, k in ((W, H), (W, H), (H, W))]
        self.shared = [I.weights(rng, o, k) for o, k in ((Wsh, H), (Wsh, H), (H, Wsh))] if Wsh else None
        self.stacks = [ctx.bind_experts([(B.K_Q8C, 8, *w) for w in p]) for p in self.parts]
        self.sh = [ctx.bind(B.K_Q8C, w[0], w[1], *w[0].shape) for w in self.shared] if Wsh else None
        self.rng = rng

    def want(self, x, idx, w):
        return I.routed(x, idx, w, *self.parts, self.shared)

    def free(self):
        for t in self.stacks + (self.sh or []):
            t.free()


def same(got, want):
    got = got.cpu().numpy()
    bad = got.view(np.uint32) != want.view(np.uint32)
    assert not (bad & ~(np.isnan(got) & np.isnan(want)) & ~((got == 0) & (want == 0))).any(), (bad.sum(), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


SHAPES = [  # E, K, H, W, Wsh, T
    (4, 1, 64, 64, 0, 1), (8, 2, 128, 192, 64, 1), (64, 6, 512, 320, 640, 1), (8, 8, 192, 128, 128, 2), (16, 3, 256, 448, 0, 3),
    (64, 6, 256, 320, 128, 4), (60, 4, 320, 1408, 704, 5), (16, 4, 128, 64, 64, 8), (33, 2, 192, 256, 0, 9), (64, 6, 320, 192, 256, 16),
    (7, 3, 64, 128, 64, 17), (64, 8, 128, 128, 128, 33), (3, 3, 128, 64, 192, 64), (2, 1, 64, 64, 0, 64), (16, 16, 64, 128, 64, 64),
    (8, 2, 64, 64, 64, 65), (16, 5, 128, 64, 0, 130), (256, 8, 64, 64, 64, 12),
    (3, 2, 16448, 64, 64, 3), (3, 2, 64, 16448, 8256, 5), (4, 2, 64, 192, 33024, 2)]


@pytest.mark.parametrize("E,K,H,W,Wsh,T", SHAPES)
def test_layer(ctx, torch_dev, E, K, H, W, Wsh, T):
    print("[case] layer", E, K, H, W, Wsh, T, flush=True)
    torch = torch_dev
    lay = Layer(ctx, [E, K, H, W, T], E, H, W, Wsh)
    x = lay.rng.standard_normal((T, H)).astype(np.float32)
    x[:, H // 2] *= 12
    rw, rb = (lay.rng.standard_normal((E, H)) / H ** 0.5).astype(np.float32), lay.rng.standard_normal(E).astype(np.float32)
    xd, rwd, rbd = (torch.from_numpy(v).cuda() for v in (x, rw, rb))
    out = torch.full((T, H), float("nan"), device="cuda")
    idx, w = torch.empty((T, K), dtype=torch.int32, device="cuda"), torch.empty((T, K), device="cuda")
    torch.cuda.synchronize()
    for bias, renorm in ((None, False), (rbd, True)):
        ctx.moe_route(rwd, xd, K, idx, w, router_b=bias, renorm=renorm)         # its own tests hold it to the oracle
        ctx.moe_layer(rwd, *lay.stacks, lay.sh, xd, K, out, router_b=bias, renorm=renorm)
        ctx.sync()
        want = lay.want(x, idx.cpu().numpy(), w.cpu().numpy())
        same(out, want)
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        ctx.moe_ffn(*lay.stacks, lay.sh, xd, idx, w, out)
        ctx.sync()
        same(out, want)
    lay.free()


@pytest.mark.parametrize("T", [1, 6, 40])
def test_given_routings(ctx, torch_dev, T):
    """One expert for all pairs, the same expert twice for a token, ids outside the stack, tokens with no expert at all."""
    torch = torch_dev
    E, K, H, W = 10, 5, 128, 192
    for Wsh in (64, 0):
        lay = Layer(ctx, [T, Wsh], E, H, W, Wsh)
        x = lay.rng.standard_normal((T, H)).astype(np.float32)
        w = lay.rng.standard_normal((T, K)).astype(np.float32)
        some = lay.rng.integers(0, E, (T, K)).astype(np.int32)
        holes = some.copy()
        holes[::2, 1] = -1
        holes[:, 3] = E
        holes[T // 2] = 2 ** 31 - 1
        for idx in (np.full((T, K), 7, np.int32), some, np.sort(some, 1)[:, ::-1].copy(), holes, np.full((T, K), -5, np.int32)):
            xd, wd, idd = (torch.from_numpy(v).cuda() for v in (x, w, idx))
            out = torch.full((T, H), float("nan"), device="cuda")
            torch.cuda.synchronize()
            ctx.moe_ffn(*lay.stacks, lay.sh, xd, idd, wd, out)
            ctx.sync()
            same(out, lay.want(x, idx, w))
        lay.free()


def test_most_experts_and_picks(ctx, torch_dev):
    """1024 experts, 16 a token, 64 tokens: as many experts as pairs."""
    torch = torch_dev
    E, K, H, W, T = 1024, 16, 64, 64, 64
    lay = Layer(ctx, 6, E, H, W, 128)
    x, w = lay.rng.standard_normal((T, H)).astype(np.float32), lay.rng.standard_normal((T, K)).astype(np.float32)
    for idx in (lay.rng.permutation(E).reshape(T, K).astype(np.int32), lay.rng.integers(0, E, (T, K)).astype(np.int32)):
        xd, wd, idd = (torch.from_numpy(v).cuda() for v in (x, w, idx))
        out = torch.full((T, H), float("nan"), device="cuda")
        torch.cuda.synchronize()
        ctx.moe_ffn(*lay.stacks, lay.sh, xd, idd, wd, out)
        ctx.check()
        same(out, lay.want(x, idx, w))
    lay.free()


def test_rows_at_the_ends_of_fp32(ctx, torch_dev):
    """A token of NaN, infinities or zeros changes no other token's bits."""
    torch = torch_dev
    E, K, H, W, T = 8, 2, 128, 64, 7
    lay = Layer(ctx, 5, E, H, W, 64)
    x = lay.rng.standard_normal((T, H)).astype(np.float32)
    x[1], x[2, 3], x[3, 4], x[4], x[5] = 0, np.nan, np.inf, x[4] * np.float32(1e-38), x[5] * np.float32(1e18)
    idx, w = lay.rng.integers(0, E, (T, K)).astype(np.int32), lay.rng.uniform(0, 1, (T, K)).astype(np.float32)
    xd, wd, idd = (torch.from_numpy(v).cuda() for v in (x, w, idx))
    out = torch.empty((T, H), device="cuda")
    torch.cuda.synchronize()
    ctx.moe_ffn(*lay.stacks, lay.sh, xd, idd, wd, out)
    ctx.sync()
    same(out, lay.want(x, idx, w))
    assert np.isnan(out[2:4].cpu().numpy()).all()
    lay.free()


@pytest.mark.parametrize("T", [1, 4, 40, 70])
@pytest.mark.parametrize("Wsh", [0, 64])
def test_scores_without_a_softmax(ctx, torch_dev, T, Wsh):
    """A token with NaN or an infinity, or whose scores are not finite for the router's own values, comes out as NaN, with and
    without shared experts and renorm; the other tokens keep their bits."""
    torch = torch_dev
    E, K, H, W = 12, 3, 128, 64
    lay = Layer(ctx, [9, Wsh], E, H, W, Wsh)
    x, rw = lay.rng.standard_normal((T, H)).astype(np.float32), (lay.rng.standard_normal((E, H)) / H ** 0.5).astype(np.float32)
    bias = lay.rng.standard_normal(E).astype(np.float32)
    idx, w, out = torch.empty((T, K), dtype=torch.int32, device="cuda"), torch.empty((T, K), device="cuda"), torch.empty((T, H), device="cuda")
    xd, rwd, bd = (torch.from_numpy(v).cuda() for v in (x, rw, bias))
    torch.cuda.synchronize()
    for renorm in (False, True):
        ctx.moe_route(rwd, xd, K, idx, w, router_b=bd, renorm=renorm)
        ctx.sync()
        want = lay.want(x, idx.cpu().numpy(), w.cpu().numpy())
        for token, place, value in ((0, H - 1, np.nan), (T // 2, 0, np.inf), (T - 1, 7, -np.inf)):
            bad = x.copy()
            bad[token, place] = value
            xb = torch.from_numpy(bad).cuda()
            out.zero_()
            torch.cuda.synchronize()
            ctx.moe_layer(rwd, *lay.stacks, lay.sh, xb, K, out, router_b=bd, renorm=renorm)
            ctx.check()
            wb = want.copy()
            wb[token] = np.nan
            same(out, wb)
        for value in (np.nan, np.inf):                      # of the router itself: every token's
            bb = torch.from_numpy(np.where(np.arange(E) == 5, np.float32(value), bias)).cuda()
            out.zero_()
            torch.cuda.synchronize()
            ctx.moe_layer(rwd, *lay.stacks, lay.sh, xd, K, out, router_b=bb, renorm=renorm)
            ctx.check()
            assert torch.isnan(out).all()
        # one expert that no token can pick (-Inf) leaves the softmax of the others
        bb = torch.from_numpy(np.where(np.arange(E) == 5, np.float32(-np.inf), bias)).cuda()
        torch.cuda.synchronize()
        ctx.moe_route(rwd, xd, K, idx, w, router_b=bb, renorm=renorm)
        ctx.moe_layer(rwd, *lay.stacks, lay.sh, xd, K, out, router_b=bb, renorm=renorm)
        ctx.check()
        assert not (idx == 5).any()
        same(out, lay.want(x, idx.cpu().numpy(), w.cpu().numpy()))
    lay.free()


@pytest.mark.parametrize("T", [1, 5, 20, 70])
def test_captured_layer(torch_dev, T):
    """Captured after one eager run and replayed on new tokens, twice into each of two graphs of one context, with eager
    calls of the same layer between."""
    import beglin_amd as B
    torch = torch_dev
    E, K, H, W = 16, 4, 256, 128
    stream = torch.cuda.Stream()
    c = B.Context(0, stream.cuda_stream)
    lays = [Layer(c, 21 + i, E, H, W, 64) for i in range(2)]
    rws = [torch.from_numpy((l.rng.standard_normal((E, H)) / H ** 0.5).astype(np.float32)).cuda() for l in lays]
    x, outs = torch.zeros((T, H), device="cuda"), [torch.empty((T, H), device="cuda") for _ in lays]
    idx, w = torch.empty((T, K), dtype=torch.int32, device="cuda"), torch.empty((T, K), device="cuda")
    torch.cuda.synchronize()
    graphs = []
    with torch.cuda.stream(stream):
        for l, r, o in zip(lays, rws, outs):
            c.moe_layer(r, *l.stacks, l.sh, x, K, o)
        stream.synchronize()
        for l, r, o in zip(lays, rws, outs):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                c.moe_layer(r, *l.stacks, l.sh, x, K, o)
            graphs.append(g)
    rng = np.random.default_rng(T)
    for i in range(3):
        xn = rng.standard_normal((T, H)).astype(np.float32)
        x.copy_(torch.from_numpy(xn))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for g in graphs + graphs[::-1]:
                g.replay()
        torch.cuda.synchronize()
        for l, r, o in zip(lays, rws, outs):
            c.moe_route(r, x, K, idx, w)
            c.sync()
            want = l.want(xn, idx.cpu().numpy(), w.cpu().numpy())
            same(o, want)
            o2 = torch.empty_like(o)
            torch.cuda.synchronize()
            c.moe_layer(r, *l.stacks, l.sh, x, K, o2)
            c.sync()
            same(o2, want)
    del graphs
    for l in lays:
        l.free()
    c.close()


def test_launches_of_changing_sizes(ctx, torch_dev):
    """Launches of many and of few workgroups after each other leave nothing behind: the same bits each time."""
    torch = torch_dev
    E, K, H, W = 24, 4, 256, 192
    lay = Layer(ctx, 77, E, H, W, 320)
    rw = torch.from_numpy((lay.rng.standard_normal((E, H)) / H ** 0.5).astype(np.float32)).cuda()
    xs = [torch.from_numpy(lay.rng.standard_normal((T, H)).astype(np.float32)).cuda() for T in (1, 64, 2, 7, 33, 1, 70, 16)]
    first = None
    for r in range(6):
        outs = [torch.full_like(x, float("nan")) for x in xs]
        torch.cuda.synchronize()
        for x, o in list(zip(xs, outs))[::1 if r % 2 else -1]:
            ctx.moe_layer(rw, *lay.stacks, lay.sh, x, K, o)
        ctx.check()
        outs = [o.cpu().numpy() for o in outs]
        if first is None:
            first = outs
            for x, o in zip(xs, outs):
                idx, w = torch.empty((len(x), K), dtype=torch.int32, device="cuda"), torch.empty((len(x), K), device="cuda")
                torch.cuda.synchronize()
                ctx.moe_route(rw, x, K, idx, w)
                ctx.sync()
                same(torch.from_numpy(o), lay.want(x.cpu().numpy(), idx.cpu().numpy(), w.cpu().numpy()))
        assert all(np.array_equal(a.view(np.uint32), b.view(np.uint32)) for a, b in zip(first, outs)), r
    lay.free()


@pytest.mark.parametrize("T", [1, 9, 40])
def test_layers_back_to_back(torch_dev, T):
    """Launches with nothing between them, in one graph, whose codes and sums lie in the same scratch: each reads its own."""
    import beglin_amd as B
    torch = torch_dev
    E, K, H, W, N = 12, 3, 512, 320, 8
    stream = torch.cuda.Stream()
    c = B.Context(0, stream.cuda_stream)
    lay = Layer(c, [8, T], E, H, W, 384)
    rw = torch.from_numpy((lay.rng.standard_normal((E, H)) / H ** 0.5).astype(np.float32)).cuda()
    xs, outs = [torch.zeros((T, H), device="cuda") for _ in range(N)], [torch.zeros((T, H), device="cuda") for _ in range(N)]
    idx, w = torch.empty((T, K), dtype=torch.int32, device="cuda"), torch.empty((T, K), device="cuda")
    torch.cuda.synchronize()

    def step():
        for x, o in zip(xs, outs):
            c.moe_layer(rw, *lay.stacks, lay.sh, x, K, o)

    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    for r in range(3):
        for x in xs:
            x.copy_(torch.from_numpy(lay.rng.standard_normal((T, H)).astype(np.float32)))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay() if r != 1 else step()
        torch.cuda.synchronize()
        c.check()
        for x, o in zip(xs, outs):
            with torch.cuda.stream(stream):
                c.moe_route(rw, x, K, idx, w)
            c.sync()
            same(o, lay.want(x.cpu().numpy(), idx.cpu().numpy(), w.cpu().numpy()))
    del graph
    lay.free()
    c.close()


def test_two_contexts_at_once(torch_dev):
    """Two contexts on streams of their own, whose launches share the CUs."""
    import beglin_amd as B
    torch = torch_dev
    E, K, H, W = 16, 4, 512, 256
    cs, lays, rws, xs = [], [], [], []
    for i in range(2):
        cs.append(B.Context(0))
        lays.append(Layer(cs[i], 90 + i, E, H, W, 256))
        rws.append(torch.from_numpy((lays[i].rng.standard_normal((E, H)) / H ** 0.5).astype(np.float32)).cuda())
        xs.append([torch.from_numpy(lays[i].rng.standard_normal((T, H)).astype(np.float32)).cuda() for T in (1, 12, 40)])
    outs = [[[torch.full_like(x, float("nan")) for x in xs[i]] for _ in range(20)] for i in range(2)]
    torch.cuda.synchronize()
    for r in range(20):
        for i in range(2):
            for x, o in zip(xs[i], outs[i][r]):
                cs[i].moe_layer(rws[i], *lays[i].stacks, lays[i].sh, x, K, o)
    for c in cs:
        c.check()
    for i in range(2):
        for j, x in enumerate(xs[i]):
            idx, w = torch.empty((len(x), K), dtype=torch.int32, device="cuda"), torch.empty((len(x), K), device="cuda")
            torch.cuda.synchronize()
            cs[i].moe_route(rws[i], x, K, idx, w)
            cs[i].sync()
            want = lays[i].want(x.cpu().numpy(), idx.cpu().numpy(), w.cpu().numpy())
            for r in range(20):
                same(outs[i][r][j], want)
    for c, l in zip(cs, lays):
        l.free()
        c.close()


@pytest.mark.parametrize("T", [1, 20])
def test_bounded_waits_give_up(torch_dev, monkeypatch, T):
    """A launch whose waits are for what is never written (set from the host, with a few polls) still ends, is reported by
    bgl_ctx_check, and leaves the context ready for the next."""
    import beglin_amd as B
    torch = torch_dev
    print("[case] bounded waits", T, flush=True)
    monkeypatch.setenv("BGL_MLP_TEST_TIMEOUT", "1")
    monkeypatch.setenv("BGL_MLP_SPIN", "64")
    c = B.Context(0)
    monkeypatch.delenv("BGL_MLP_TEST_TIMEOUT")
    monkeypatch.delenv("BGL_MLP_SPIN")
    E, K, H, W = 16, 4, 256, 128
    lay = Layer(c, 41, E, H, W, 64)
    x = lay.rng.standard_normal((T, H)).astype(np.float32)
    xd, out = torch.from_numpy(x).cuda(), torch.empty((T, H), device="cuda")
    idx, w = lay.rng.integers(0, E, (T, K)).astype(np.int32), lay.rng.uniform(0, 1, (T, K)).astype(np.float32)
    idd, wd = torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda()
    torch.cuda.synchronize()
    c.moe_ffn(*lay.stacks, lay.sh, xd, idd, wd, out)
    with pytest.raises(B.BglError) as e:
        c.check()
    assert e.value.code == B.E_TIMEOUT
    c.check()                                             # the flag was cleared
    for _ in range(2):
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        c.moe_ffn(*lay.stacks, lay.sh, xd, idd, wd, out)
        c.check()
        same(out, lay.want(x, idx, w))
    lay.free()
    c.close()


@pytest.mark.parametrize("T", [1, 20, 70])
def test_a_layer_after_one_that_gave_up(torch_dev, monkeypatch, T):
    """The layers after one in whose odd workgroups the waits gave up (so that they saw another routing than the even ones, and
    counted other blocks) are right without a check between."""
    import beglin_amd as B
    torch = torch_dev
    print("[case] after a wait that gave up", T, flush=True)
    monkeypatch.setenv("BGL_MLP_TEST_TIMEOUT", "1")
    monkeypatch.setenv("BGL_MLP_SPIN", "2048")             # polls of the good layers too: some ms, of which they need one hundredth
    c = B.Context(0)
    monkeypatch.delenv("BGL_MLP_TEST_TIMEOUT")
    monkeypatch.delenv("BGL_MLP_SPIN")
    E, K, H, W = 16, 4, 256, 128
    lay = Layer(c, 42, E, H, W, 64)
    rw = torch.from_numpy((lay.rng.standard_normal((E, H)) / H ** 0.5).astype(np.float32)).cuda()
    xs = [lay.rng.standard_normal((T, H)).astype(np.float32) for _ in range(3)]
    outs = [torch.full((T, H), float("nan"), device="cuda") for _ in xs]
    xd = [torch.from_numpy(x).cuda() for x in xs]
    idx, w = torch.empty((T, K), dtype=torch.int32, device="cuda"), torch.empty((T, K), device="cuda")
    torch.cuda.synchronize()
    c.moe_layer(rw, *lay.stacks, lay.sh, xd[0], K, outs[0])       # (its first 64 tokens give up)
    for x, o in zip(xd[1:], outs[1:]):
        c.moe_layer(rw, *lay.stacks, lay.sh, x, K, o)
    c.sync()
    for i in (1, 2):
        c.moe_route(rw, xd[i], K, idx, w)
        c.sync()
        same(outs[i], lay.want(xs[i], idx.cpu().numpy(), w.cpu().numpy()))
    with pytest.raises(B.BglError) as e:
        c.check()
    assert e.value.code == B.E_TIMEOUT
    lay.free()
    c.close()


def test_refusals(ctx, torch_dev):
    import beglin_amd as B
    torch = torch_dev
    E, H, W = 4, 64, 64
    lay = Layer(ctx, 1, E, H, W, 64)
    rng = np.random.default_rng(0)
    other = ctx.experts_from_tensors([ctx.quantize(B.K_Q8G64, torch.randn((W, H), device="cuda")) for _ in range(E)])
    mixed = ctx.experts_from_tensors([ctx.quantize(B.K_Q8C if e else B.K_Q8G64, torch.randn((W, H), device="cuda")) for e in range(E)])
    sh8 = [ctx.quantize(B.K_Q8G64, torch.randn((64, 64), device="cuda")) for _ in range(3)]
    x, out = torch.zeros((2, H), device="cuda"), torch.full((2, H), 3.0, device="cuda")
    idx, w, rw = torch.zeros((2, 2), dtype=torch.int32, device="cuda"), torch.zeros((2, 2), device="cuda"), torch.zeros((E, H), device="cuda")
    g, u, d = lay.stacks

    def refused(code, fn):
        with pytest.raises(B.BglError) as e:
            fn()
        assert e.value.code == code, e.value

    for stacks, sh in (([g, u, other], None), ([g, other, d], None), ([other, other, d], None), ([mixed, mixed, mixed], None),
                       ([g, u, d], sh8), ([other, other, other], lay.sh)):
        want = B.E_ARG if stacks[0] is not stacks[1] and other in stacks[:2] else B.E_UNSUPPORTED
        refused(want, lambda: ctx.moe_ffn(*stacks, sh, x, idx, w, out))
        refused(want, lambda: ctx.moe_layer(rw, *stacks, sh, x, 2, out))
    refused(B.E_ARG, lambda: ctx.moe_layer(rw, g, u, d, None, x, 5, out))                      # more picks than experts
    refused(B.E_UNSUPPORTED, lambda: ctx.gather_matvec(g, x, idx[:, 0].contiguous(), out))
    ctx.sync()
    assert torch.equal(out.cpu(), torch.full((2, H), 3.0))
    for t in [other, mixed] + sh8:
        t.free()
    lay.free()
