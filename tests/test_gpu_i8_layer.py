"""Two transformer layers' projections of int8 weights as a decoder runs them, in one captured graph: norm to codes, the q / k / v
products of the codes, an output product of fp32 rows, the residual add with the next norm, an MLP or a routed layer, and the
last norm into the output head.  (The attention between them is not this library's: v stands for what it gives.)  Every step
is checked from the inputs that it found on the device, bit for bit where the sums are exact."""
import numpy as np
import pytest

import int8_forms as I

pytestmark = pytest.mark.gpu

H, W, E, K, WE = 320, 448, 8, 2, 192


@pytest.fixture(scope="module")
def torch_dev():
    import torch
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    return torch


def near(got, want, name):
    """fp32 values of the 64-bit formula: half a step of rounding, and what doubles are off by before it."""
    off = np.abs(got.astype(np.float64) - want) - np.abs(want) * (2.0 ** -24 * (1 + 1e-6)) - 1e-45
    assert off.max() <= 0, (name, off.max())


@pytest.mark.parametrize("T", [1, 5, 70])
def test_two_layers(torch_dev, T):
    import beglin_amd as B
    torch = torch_dev
    print("[case] layers", T, flush=True)
    rng = np.random.default_rng(T)
    stream = torch.cuda.Stream()
    c = B.Context(0, stream.cuda_stream)
    dev = lambda v: torch.from_numpy(v).cuda()  # noqa: E731
    new = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt, device="cuda")  # noqa: E731
    bind = lambda w: c.bind(B.K_Q8C, w[0], w[1], *w[0].shape)  # noqa: E731
    qkv = [[I.weights(rng, n, H) for n in (H, 64, 64)] for _ in range(2)]
    wo = [I.weights(rng, H, H) for _ in range(2)]
    mlp = [I.weights(rng, W, H), I.weights(rng, W, H), I.weights(rng, H, W)]
    exp = [[I.weights(rng, o, k) for _ in range(E)] for o, k in ((WE, H), (WE, H), (H, WE))]
    sh = [I.weights(rng, o, k) for o, k in ((64, H), (64, H), (H, 64))]
    head = I.weights(rng, 1000, H)
    router = (rng.standard_normal((E, H)) / H ** 0.5).astype(np.float32)
    norms = (1 + 0.1 * rng.standard_normal((5, H))).astype(np.float32)
    t_qkv, t_wo, t_mlp, t_sh, t_head = [[bind(w) for w in p] for p in qkv], [bind(w) for w in wo], [bind(w) for w in mlp], [bind(w) for w in sh], bind(head)
    t_exp = [c.bind_experts([(B.K_Q8C, 8, *w) for w in p]) for p in exp]
    nd, rd = [dev(v) for v in norms], dev(router)
    x = new(T, H)
    res = [new(T, H) for _ in range(5)]                    # the residual rows after each add
    ns = [new(T, H) for _ in range(5)]
    qs, ss = [new(T, H, dt=torch.int8) for _ in range(3)], [new(T) for _ in range(3)]
    qv = [[new(T, w[0].shape[0]) for w in p] for p in qkv]
    att, ffn, logits = [new(T, H) for _ in range(2)], [new(T, H) for _ in range(2)], new(T, 1000, dt=torch.bfloat16)
    idx, wt = new(T, K, dt=torch.int32), new(T, K)

    def step():
        c.norm(x, y=ns[0], yq=qs[0], yscale=ss[0], w=nd[0], x_out=res[0])
        c.matmul_i8(t_qkv[0], qs[0], ss[0], qv[0])
        c.matmul(t_wo[0], qv[0][0], att[0], act=B.ACT_W4A8)
        c.norm(res[0], y=ns[1], w=nd[1], x_out=res[1], branch=att[0])
        c.mlp(*t_mlp, ns[1], ffn[0], act=B.ACT_W4A8)
        c.norm(res[1], y=ns[2], yq=qs[1], yscale=ss[1], w=nd[2], x_out=res[2], branch=ffn[0])
        c.matmul_i8(t_qkv[1], qs[1], ss[1], qv[1])
        c.matmul(t_wo[1], qv[1][0], att[1], act=B.ACT_W4A8)
        c.norm(res[2], y=ns[3], w=nd[3], x_out=res[3], branch=att[1])
        c.moe_layer(rd, *t_exp, t_sh, ns[3], K, ffn[1], renorm=True)
        c.norm(res[3], y=ns[4], yq=qs[2], yscale=ss[2], w=nd[4], x_out=res[4], branch=ffn[1])
        c.matmul_i8(t_head, qs[2], ss[2], logits)

    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    for r in range(4):
        x.copy_(dev(rng.standard_normal((T, H)).astype(np.float32)))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay() if r else step()
        torch.cuda.synchronize()
        c.check()
        h = lambda t: t.cpu().numpy()  # noqa: E731
        same = lambda got, want: np.array_equal(got.view(np.uint32), np.asarray(want, np.float32).view(np.uint32))  # noqa: E731
        rows = [h(v) for v in res]
        assert same(rows[0], h(x))
        for i, b in ((1, att[0]), (2, ffn[0]), (3, att[1]), (4, ffn[1])):
            assert same(rows[i], rows[i - 1] + h(b)), i
        for i, n in enumerate(ns):
            near(h(n), I.normed(1, rows[i], norms[i]), i)
        for i, j in ((0, 0), (1, 2), (2, 4)):
            q, s = I.quantize(h(ns[j]))
            assert np.array_equal(h(qs[i]), q) and same(h(ss[i]), s), i
        for i in range(2):
            for got, w in zip(qv[i], qkv[i]):
                assert same(h(got), I.product(h(qs[i]), h(ss[i]), *w))
            assert same(h(att[i]), I.product(*I.quantize(h(qv[i][0])), *wo[i]))
        assert same(h(ffn[0]), I.mlp(h(ns[1]), *mlp)[1])
        with torch.cuda.stream(stream):
            c.moe_route(rd, ns[3], K, idx, wt, renorm=True)
        c.sync()
        assert same(h(ffn[1]), I.routed(h(ns[3]), h(idx), h(wt), *exp, sh))
        assert torch.equal(logits.cpu(), torch.from_numpy(I.product(h(qs[2]), h(ss[2]), *head)).bfloat16())
        _ = (x * 2).sum().item()                           # eager work of the program's own
    del graph
    for t in sum(t_qkv, []) + t_wo + t_mlp + t_sh + t_exp + [t_head]:
        t.free()
    c.close()
