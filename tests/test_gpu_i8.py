"""int8 products with one scale per token and per output channel (K_Q8C) against the plain numpy form, bit for bit: the
sum of codes is exact in both, and every fp32 step after it is one rounded operation."""
import numpy as np
import pytest

import int8_forms as I

pytestmark = pytest.mark.gpu


def say(*a):
    print("[case]", *a, flush=True)


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


def bind(ctx, w):
    import beglin_amd as B
    return ctx.bind(B.K_Q8C, w[0], w[1], *w[0].shape)


def same(got, want):
    got = got.cpu().numpy()
    assert got.shape == want.shape and got.dtype == want.dtype
    bad = got.view(np.uint32) != want.view(np.uint32)
    assert not (bad & ~(np.isnan(got) & np.isnan(want))).any(), (bad.sum(), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


def codes(torch, rng, M, K, pad=0):
    """Codes as the library's calls take them: rows a multiple of 16 bytes apart, anything behind each row."""
    ld = (K + 15) // 16 * 16 + 16 * pad
    q = rng.integers(-128, 128, (M, ld)).astype(np.int8)
    s = rng.uniform(0.005, 0.03, M).astype(np.float32)
    return q, s, torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda()


# tokens around each launch's column blocks, channels around 16 / 64 / 256, K around 16, 64 and 128
SHAPES = [(1, 1, 1), (1, 64, 64), (1, 8960, 1536), (2, 17, 100), (3, 63, 127), (5, 65, 128), (16, 256, 129), (17, 1001, 1411),
          (31, 15, 16), (33, 4096, 500), (48, 130, 4096), (49, 9000, 192), (64, 1024, 14336), (64, 33000, 80), (12, 40000, 256),
          (20, 33000, 128), (65, 64, 64), (65, 1, 1), (100, 257, 255), (128, 512, 256), (129, 300, 1000), (255, 255, 384),
          (256, 256, 4096), (257, 1030, 640), (333, 1001, 1411), (1000, 96, 2048), (640, 2600, 512), (2049, 520, 272), (1500, 6144, 1024),
          (1411, 6001, 1090)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_of_codes(ctx, torch_dev, M, N, K):
    say("codes", M, N, K)
    rng = np.random.default_rng([M, N, K])
    w = I.weights(rng, N, K)
    b = rng.standard_normal(N).astype(np.float32)
    q, s, qd, sd = codes(torch_dev, rng, M, K, pad=M % 3)
    t, y = bind(ctx, w), torch_dev.full((M, N), float("nan"), device="cuda")
    torch_dev.cuda.synchronize()
    ctx.matmul_i8(t, qd, sd, y)
    ctx.sync()
    same(y, I.product(q[:, :K], s, *w))
    ctx.matmul_i8(t, qd, sd, y, torch_dev.from_numpy(b).cuda())
    ctx.sync()
    same(y, I.product(q[:, :K], s, *w, b))
    t.free()


@pytest.mark.parametrize("M", [1, 40, 70, 300])
@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
def test_16_bit_outputs_round_the_fp32_value(ctx, torch_dev, M, kind):
    N, K = 330, 700
    rng = np.random.default_rng(M)
    w = I.weights(rng, N, K)
    q, s, qd, sd = codes(torch_dev, rng, M, K)
    t, y = bind(ctx, w), torch_dev.zeros((M, N), dtype=getattr(torch_dev, kind), device="cuda")
    torch_dev.cuda.synchronize()
    ctx.matmul_i8(t, qd, sd, y)
    ctx.sync()
    want = torch_dev.from_numpy(I.product(q[:, :K], s, *w)).to(y.dtype)
    assert torch_dev.equal(y.cpu(), want)
    t.free()


@pytest.mark.parametrize("M", [1, 9, 64, 65, 200])
def test_group_fills_the_parts_of_wider_rows(ctx, torch_dev, M):
    """q, k and v side by side in one row, with room left between and behind, and other values there kept."""
    rng = np.random.default_rng(M)
    K, parts = 384, [(0, 200), (203, 64), (270, 33)]
    ws = [I.weights(rng, n, K) for _, n in parts]
    bs = [rng.standard_normal(n).astype(np.float32) if i != 1 else None for i, (_, n) in enumerate(parts)]
    q, s, qd, sd = codes(torch_dev, rng, M, K)
    ts = [bind(ctx, w) for w in ws]
    row = torch_dev.full((M, 311), 7.0, device="cuda")
    bd = [torch_dev.from_numpy(b).cuda() if b is not None else None for b in bs]
    torch_dev.cuda.synchronize()
    ctx.matmul_i8(ts, qd, sd, [row[:, a:a + n] for a, n in parts], bd)
    ctx.sync()
    want = np.full((M, 311), 7.0, np.float32)
    for (a, n), w, b in zip(parts, ws, bs):
        want[:, a:a + n] = I.product(q[:, :K], s, *w, b)
    same(row, want)
    for t in ts:
        t.free()


@pytest.mark.parametrize("M,rows,K", [(1, [300], 1536), (4, [70, 33], 96), (7, [64, 64, 64, 64], 130), (64, [500], 1000),
                                      (65, [129], 4099), (130, [90, 600], 257), (3, [40], 20000)])
def test_fp32_columns(ctx, torch_dev, M, rows, K):
    """matmul / matmul_group quantize each column by its own largest value."""
    say("columns", M, rows, K)
    rng = np.random.default_rng([M, K])
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[:, K // 3] *= 40
    x[M // 2] *= np.float32(1e-30)
    ws = [I.weights(rng, n, K) for n in rows]
    bs = [rng.standard_normal(n).astype(np.float32) if i % 2 else None for i, n in enumerate(rows)]
    ts, xd = [bind(ctx, w) for w in ws], torch_dev.from_numpy(x).cuda()
    ys = [torch_dev.empty((M, n), device="cuda") for n in rows]
    bd = [torch_dev.from_numpy(b).cuda() if b is not None else None for b in bs]
    torch_dev.cuda.synchronize()
    ctx.matmul_group(ts, xd, ys, act=1, biases=bd)
    ctx.sync()
    q, s = I.quantize(x)
    for y, w, b in zip(ys, ws, bs):
        same(y, I.product(q, s, *w, b))
    # prepared once, used for fewer columns too, and without the allocating scratch
    y = torch_dev.empty((M, rows[0]), device="cuda")
    ctx.prep_only(xd, 1, ts[0])
    ctx.matmul_prepped(ts[0], y, act=1, M=M)
    ctx.sync()
    same(y, I.product(q, s, *ws[0]))
    for t in ts:
        t.free()


@pytest.mark.parametrize("M,rows,K", [(1, [64], 64), (1, [300, 70], 8192), (1, [17], 16384), (1, [4000], 16320), (2, [130], 4096), (8, [33, 900], 1024),
                                      (16, [40], 512), (15, [65, 1], 448), (3, [500], 2688), (5, [9000], 1600), (2, [20, 20, 20, 20], 4032)])
def test_few_fp32_columns(ctx, torch_dev, M, rows, K):
    """Few values, whose codes each workgroup makes (K whole and split): the bits of quantizing first, also where the columns
    begin off 16 bytes, and rows of NaN, infinities, zeros."""
    say("few columns", M, rows, K)
    rng = np.random.default_rng([M, K, 7])
    ws, bs = [I.weights(rng, n, K) for n in rows], [rng.standard_normal(n).astype(np.float32) for n in rows]
    ts, bd = [bind(ctx, w) for w in ws], [torch_dev.from_numpy(b).cuda() for b in bs]
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[:, K // 3] *= 40
    wild = x.copy()
    wild[0, K - 1] = np.nan
    wild[M // 2, 3] = -np.inf
    for v in (x, wild, np.zeros_like(x)):
        for off in (0, 1, 3):
            xd = torch_dev.zeros(M * K + 8, device="cuda")[off:off + M * K].view(M, K)
            xd.copy_(torch_dev.from_numpy(v))
            ys = [torch_dev.empty((M, n), device="cuda") for n in rows]
            torch_dev.cuda.synchronize()
            ctx.matmul_group(ts, xd, ys, act=1, biases=bd)
            ctx.sync()
            q, s = I.quantize(v)
            for y, w, b in zip(ys, ws, bs):
                same(y, I.product(q, s, *w, b))
    for t in ts:
        t.free()


@pytest.mark.parametrize("M", [1, 20, 64, 200])
def test_split_sums_are_joined(ctx, torch_dev, M):
    """Few channels and a long K, which several workgroups share: groups, biases, strided 16-bit rows, then fewer columns in
    a graph after the larger eager call."""
    say("split K", M)
    torch = torch_dev
    rng = np.random.default_rng(M)
    K, rows = 9000, [70, 5, 130]
    ws, bs = [I.weights(rng, n, K) for n in rows], [rng.standard_normal(rows[0]).astype(np.float32), None, rng.standard_normal(rows[2]).astype(np.float32)]
    import beglin_amd as B
    stream = torch.cuda.Stream()
    c = B.Context(0, stream.cuda_stream)
    ts = [bind(c, w) for w in ws]
    bd = [torch.from_numpy(b).cuda() if b is not None else None for b in bs]
    q, s, qd, sd = codes(torch, rng, M, K)
    for dt in (torch.float32, torch.bfloat16):
        wide = torch.full((M, 301), 7.0, dtype=dt, device="cuda")
        ys = [wide[:, 1:71], wide[:, 80:85], wide[:, 100:230]]
        torch.cuda.synchronize()
        c.matmul_i8(ts, qd, sd, ys, biases=bd)
        c.sync()
        want = torch.full((M, 301), 7.0)
        for at, w, b in zip((1, 80, 100), ws, bs):
            want[:, at:at + w[0].shape[0]] = torch.from_numpy(I.product(q[:, :K], s, *w, b))
        assert torch.equal(wide.cpu(), want.to(dt))
    m = (M + 1) // 2
    y = torch.empty((m, rows[2]), device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            c.matmul_i8(ts[2], qd[:m], sd[:m], y)
    for r in range(3):
        y.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
            c.matmul_i8(ts[0], qd, sd, torch.empty((M, rows[0]), device="cuda"))       # eager work that uses the same sums
        torch.cuda.synchronize()
        same(y, I.product(q[:m, :K], s[:m], *ws[2]))
    del graph
    for t in ts:
        t.free()
    c.close()


def test_columns_at_the_ends_of_fp32(ctx, torch_dev):
    """Zeros, subnormals, 1e38, infinities and NaN: a row that holds one of the last two gives NaN, the others nothing of it."""
    rng = np.random.default_rng(3)
    M, N, K = 9, 80, 200
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e-40)
    x[2] *= np.float32(1e37)
    x[3, 5], x[4, 7], x[5, 9], x[5, 10] = np.inf, -np.inf, np.nan, np.inf
    x[6] = -0.0
    w = I.weights(rng, N, K)
    t, xd, y = bind(ctx, w), torch_dev.from_numpy(x).cuda(), torch_dev.empty((M, N), device="cuda")
    torch_dev.cuda.synchronize()
    ctx.matmul(t, xd, y, act=1)
    ctx.sync()
    same(y, I.product(*I.quantize(x), *w))
    assert np.isnan(y[3:6].cpu().numpy()).all() and np.isfinite(np.delete(y.cpu().numpy(), [3, 4, 5], 0)).all()
    t.free()


def test_largest_sums(ctx, torch_dev):
    """Every product 128 * 128 over the longest K: the int32 sum reaches 2147467264 and does not wrap."""
    K, N, M = 131071, 20, 3
    w = (np.full((N, K), -128, np.int8), np.full(N, 1e-3, np.float32))
    q = np.full((M, K + 1), -128, np.int8)
    s = np.array([1e-2, 1.0, 3.0], np.float32)
    for M2 in (M, 70):
        q2, s2 = np.resize(q, (M2, K + 1)), np.resize(s, M2)
        t, y = bind(ctx, w), torch_dev.empty((M2, N), device="cuda")
        ctx.matmul_i8(t, torch_dev.from_numpy(q2).cuda(), torch_dev.from_numpy(s2).cuda(), y)
        ctx.sync()
        same(y, I.product(q2[:, :K], s2, *w))
        t.free()


@pytest.mark.parametrize("out,inn", [(1, 1), (64, 128), (77, 100), (130, 1411), (200, 4096), (9, 17000)])
def test_bind_decode_and_quantize(ctx, torch_dev, out, inn):
    import beglin_amd as B
    rng = np.random.default_rng([out, inn])
    w = I.weights(rng, out, inn)
    t = bind(ctx, w)
    info = t.info()
    assert (info["kind"], info["bits"], info["out"], info["inn"]) == (B.K_Q8C, 8, out, inn)
    d = torch_dev.empty((out, inn), device="cuda")
    ctx.dequant(t, 0, out, d)
    ctx.sync()
    same(d, w[0].astype(np.float32) * w[1][:, None])
    t.free()
    dense = rng.standard_normal((out, inn)).astype(np.float32)
    t, (pk, sc, sub) = ctx.quantize(B.K_Q8C, torch_dev.from_numpy(dense).cuda(), want_ref=True)
    q, s = I.quantize(dense)
    assert sub is None and np.array_equal(pk, q) and np.array_equal(sc.view(np.uint32), s.view(np.uint32))
    ctx.dequant(t, 0, out, d)
    ctx.sync()
    same(d, q.astype(np.float32) * s[:, None])
    t.free()


@pytest.mark.parametrize("kind,bits", [("K_Q8C", 8), ("K_Q4G64", 4), ("K_Q8G64", 8), ("K_QNG64", 5), ("K_Q4G32H", 4), ("K_Q4G256SF", 4)])
def test_bind_from_the_device(ctx, torch_dev, kind, bits):
    """Weights that are on the device are bound from there, aligned or not, to the same tensor as from the host; the buffers are
    the caller's again when the call returns."""
    import beglin_amd as B
    torch = torch_dev
    kind = getattr(B, kind)
    for out, inn in ((77, 100), (130, 1411), (64, 512)) if kind == B.K_Q8C else ((70, 512),):
        dense = torch.from_numpy(np.random.default_rng([out, inn]).standard_normal((out, inn)).astype(np.float32)).cuda()
        torch.cuda.synchronize()
        t0, ref = ctx.quantize(kind, dense, bits=bits, want_ref=True)
        t0.free()
        got = []
        for off in (None, 0, 1, 8):                          # from the host; on the device, codes at any address
            bufs = list(ref)
            if off is not None:
                for i, v in enumerate(ref):
                    if v is not None:
                        dt = torch.int8 if i != 1 else torch.float16 if kind == B.K_Q4G32H else torch.float32
                        at = off if i == 0 else 16
                        raw = torch.zeros(v.nbytes + 64, dtype=torch.uint8, device="cuda")[at:at + v.nbytes]
                        raw.copy_(torch.from_numpy(np.frombuffer(v.tobytes(), np.uint8).copy()))
                        bufs[i] = raw.view(dt)
            torch.cuda.synchronize()
            t = ctx.bind(kind, bufs[0], bufs[1], out, inn, bits=bits, sub=bufs[2])
            if off is not None:
                for v in bufs:
                    if v is not None:
                        v.zero_()
                torch.cuda.synchronize()
            d = torch.full((out, inn), float("nan"), device="cuda")
            torch.cuda.synchronize()
            ctx.dequant(t, 0, out, d)
            ctx.sync()
            got.append(d.cpu().numpy())
            t.free()
        assert np.isfinite(got[0]).all()
        for g in got[1:]:
            assert np.array_equal(g.view(np.uint32), got[0].view(np.uint32))


def test_experts_from_the_device(ctx, torch_dev):
    import beglin_amd as B
    torch = torch_dev
    rng = np.random.default_rng(12)
    E, K, H, W, T = 5, 2, 64, 128, 6
    parts = [[I.weights(rng, o, k) for _ in range(E)] for o, k in ((W, H), (W, H), (H, W))]
    on = [[tuple(torch.from_numpy(v).cuda() for v in w) for w in p] for p in parts]
    torch.cuda.synchronize()
    stacks = [ctx.bind_experts([(B.K_Q8C, 8, *w) for w in p]) for p in on]
    x, idx, w = rng.standard_normal((T, H)).astype(np.float32), rng.integers(0, E, (T, K)).astype(np.int32), rng.uniform(0, 1, (T, K)).astype(np.float32)
    out, xd, idd, wd = torch.empty((T, H), device="cuda"), *(torch.from_numpy(v).cuda() for v in (x, idx, w))
    torch.cuda.synchronize()
    ctx.moe_ffn(*stacks, None, xd, idd, wd, out)
    ctx.check()
    same(out, I.routed(x, idx, w, *parts))
    for t in stacks:
        t.free()


@pytest.mark.parametrize("M,H,W", [(1, 256, 700), (5, 96, 130), (33, 1000, 333), (64, 512, 2048), (90, 300, 1001), (2, 64, 18000)])
def test_mlp(ctx, torch_dev, M, H, W):
    rng = np.random.default_rng([M, H, W])
    x = rng.standard_normal((M, H)).astype(np.float32)
    g, u, d = I.weights(rng, W, H), I.weights(rng, W, H), I.weights(rng, H, W)
    ts = [bind(ctx, w) for w in (g, u, d)]
    y, h = torch_dev.empty((M, H), device="cuda"), torch_dev.empty((M, W), device="cuda")
    xd = torch_dev.from_numpy(x).cuda()
    torch_dev.cuda.synchronize()
    ctx.mlp(*ts, xd, y, act=1, h_dev=h)
    ctx.sync()
    wh, wy = I.mlp(x, g, u, d)
    # exp in double may differ by its last bit between this host's and the device's: h by an fp32 rounding
    # where that crosses a border (about 1 value in 2^29); none at these sizes and seeds
    same(h, wh)
    same(y, wy)
    y2 = torch_dev.empty_like(y)
    ctx.mlp(*ts, xd, y2, act=1)
    ctx.sync()
    same(y2, wy)
    for t in ts:
        t.free()


@pytest.mark.parametrize("M", [3, 150])
def test_captured_call(ctx, torch_dev, M):
    """A step of group, MLP and caller-quantized product, captured after one eager run and replayed on new inputs, with
    eager work between the replays."""
    import beglin_amd as B
    torch = torch_dev
    rng = np.random.default_rng(M)
    K, W = 320, 500
    ws = [I.weights(rng, n, k) for n, k in ((200, K), (72, K), (W, K), (W, K), (K, W))]
    stream = torch.cuda.Stream()
    c = B.Context(0, stream.cuda_stream)
    ts = [bind(c, w) for w in ws]
    x = torch.empty((M, K), device="cuda")
    ys = [torch.empty((M, n), device="cuda") for n in (200, 72)]
    y, z = torch.empty((M, K), device="cuda"), torch.empty((M, 200), dtype=torch.float16, device="cuda")
    xq, xs = torch.empty((M, K), dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")

    def step():
        c.matmul_group(ts[:2], x, ys, act=1)
        c.mlp(*ts[2:], x, y, act=1)
        c.norm(y, yq=xq, yscale=xs, kind=B.NORM_NONE)
        c.matmul_i8(ts[0], xq, xs, z)

    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        x.zero_()
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    for i in range(4):
        xn = rng.standard_normal((M, K)).astype(np.float32) * np.float32(10.0 ** i)
        x.copy_(torch.from_numpy(xn))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        q, s = I.quantize(xn)
        for got, w in zip(ys, ws):
            same(got, I.product(q, s, *w))
        wy = I.mlp(xn, *ws[2:])[1]
        same(y, wy)
        want = I.product(*I.quantize(wy), *ws[0])
        assert torch.equal(z.cpu(), torch.from_numpy(want).half())
        _ = (x * 2).sum().item()
    del graph
    for t in ts:
        t.free()
    c.close()


@pytest.mark.parametrize("M,N,K", [(70000, 33000, 64), (70000, 64, 65536)])
def test_rows_past_4_gib(ctx, torch_dev, M, N, K):
    """Outputs, then codes, of more than 2^32 bytes."""
    say("past 4 GiB", M, N, K)
    torch = torch_dev
    rng = np.random.default_rng(N)
    w = I.weights(rng, N, K)
    t, y = bind(ctx, w), torch.full((M, N), 9.0, dtype=torch.float16, device="cuda")
    q, s = torch.zeros((M, K), dtype=torch.int8, device="cuda"), torch.full((M,), 0.01, device="cuda")
    some = np.array([0, 1, 32768, 65535, 65536, M - 1])
    part = rng.integers(-20, 21, (len(some), K)).astype(np.int8)
    q[torch.from_numpy(some).cuda()] = torch.from_numpy(part).cuda()
    torch.cuda.synchronize()
    ctx.matmul_i8(t, q, s, y)
    ctx.sync()
    want = torch.from_numpy(I.product(part, np.full(len(some), 0.01, np.float32), *w)).half()
    assert torch.equal(y[torch.from_numpy(some).cuda()].cpu(), want)
    assert int((y != 0).any(1).sum()) == len(some)
    t.free()


def test_noalloc(ctx, torch_dev):
    import ctypes as C

    import beglin_amd as B
    rng = np.random.default_rng(8)
    M, N, K = 20, 300, 640
    w = I.weights(rng, N, K)
    x = rng.standard_normal((M, K)).astype(np.float32)
    t, xd, y = bind(ctx, w), torch_dev.from_numpy(x).cuda(), torch_dev.empty((M, N), device="cuda")
    torch_dev.cuda.synchronize()
    W, Y, Bi = (C.c_void_p * 1)(t.h.value), (C.c_void_p * 1)(y.data_ptr()), (C.c_void_p * 1)(None)
    assert B.lib().bgl_matmul_group_noalloc_dev(ctx.h, 1, W, 1, C.c_void_p(xd.data_ptr()), Bi, Y, M) == 0
    ctx.sync()
    same(y, I.product(*I.quantize(x), *w))
    t.free()


def test_refusals(ctx, torch_dev):
    import beglin_amd as B
    torch = torch_dev
    rng = np.random.default_rng(1)
    t, other = bind(ctx, I.weights(rng, 40, 96)), bind(ctx, I.weights(rng, 40, 80))
    x, y = torch.zeros((2, 96), device="cuda"), torch.full((2, 40), 5.0, device="cuda")
    q, s = torch.zeros((2, 96), dtype=torch.int8, device="cuda"), torch.ones(2, device="cuda")
    q8 = torch.zeros((2, 64), dtype=torch.int8, device="cuda")
    int4 = ctx.quantize(B.K_Q4G64, torch.randn((40, 64), device="cuda"))

    def refused(code, fn):
        with pytest.raises(B.BglError) as e:
            fn()
        assert e.value.code == code, e.value

    refused(B.E_UNSUPPORTED, lambda: ctx.matmul(t, x, y, act=B.ACT_F32))
    refused(B.E_ARG, lambda: ctx.matmul_group([t, other], x, [y, y], act=1))
    refused(B.E_ARG, lambda: ctx.matmul_i8([t, other], q, s, [y, y]))
    refused(B.E_UNSUPPORTED, lambda: ctx.matmul_i8(int4, q8, s, y))
    refused(B.E_ARG, lambda: ctx.matmul_i8(t, q8, s, y))                                       # rows too short
    refused(B.E_ARG, lambda: ctx.matmul_i8(t, torch.zeros(2 * 100 + 8, dtype=torch.int8, device="cuda")[:200].view(2, 100), s, y))
    refused(B.E_ARG, lambda: ctx.matmul_i8(t, torch.zeros(2 * 96 + 8, dtype=torch.int8, device="cuda")[8:].view(2, 96), s, y))
    refused(B.E_ARG, lambda: ctx.matmul_prepped(t, y, act=1, M=2))                              # nothing prepared
    refused(B.E_UNSUPPORTED, lambda: ctx.prep_only(x, B.ACT_F32, t))
    refused(B.E_ARG, lambda: ctx.quant_act_i8(x, 48, q, s))
    one = np.ones(1, np.float32)
    refused(B.E_ARG, lambda: ctx.bind(B.K_Q8C, np.zeros((1, 131072), np.int8), one, 1, 131072))
    refused(B.E_ARG, lambda: ctx.bind(B.K_Q8C, np.zeros((1, 16), np.int8), None, 1, 16))
    refused(B.E_ARG, lambda: ctx.bind(B.K_Q8C, np.zeros((1, 16), np.int8), one, 1, 0))
    ctx.sync()
    assert torch.equal(y.cpu(), torch.full((2, 40), 5.0))
    for v in (t, other, int4):
        v.free()
