"""bgl_norm_dev against the formulas in 64 bits.

The kernel computes in double and rounds once to fp32 and from there to the output's type, so a value may be off by half
a step of each rounding: 2^-24, and 2^-11 (fp16) or 2^-8 (bf16) more, relative (fp16 below its normal range: half of
2^-24 absolute), plus what the order of a double sum moves (1e-12 is far above it)."""
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


def host(t):
    return t.float().cpu().numpy()


def near(got, want, name):
    """got (a tensor of its type) against 64-bit values."""
    bound = {"float32": (2.0 ** -24, 0.0), "float16": (2.0 ** -24 + 2.0 ** -11, 2.0 ** -25), "bfloat16": (2.0 ** -24 + 2.0 ** -8, 0.0)}
    rel, least = bound[str(got.dtype).split(".")[1]]
    g = host(got).astype(np.float64)
    off = np.abs(g - want) - (rel * np.abs(want) * (1 + 1e-6) + least + 1e-12 * np.abs(want) + 1e-45)
    assert np.isfinite(g).all() and off.max() <= 0, (name, off.max(), np.argwhere(off > 0)[:4])


def rows(torch, rng, T, H, kind, scale=1.0, pad=0):
    t = torch.from_numpy((rng.standard_normal((T, H + pad)) * scale).astype(np.float32)).to(getattr(torch, kind)).cuda()
    return t[:, :H]


CASES = [  # T, H, x, f, post, pre, gate, out, padding behind each row, w_add
    (1, 4096, "float32", None, 0, 1, None, "float32", 0, 0.0),
    (1, 1, "float32", "float32", 1, 1, "token", "float32", 0, 0.0),
    (3, 7, "float16", "bfloat16", 2, 2, "channel", "float16", 0, 0.0),
    (33, 64, "bfloat16", "bfloat16", 0, 1, None, "bfloat16", 0, 1.0),
    (5, 1000, "float32", "float16", 1, 1, "full", "float32", 24, 1.0),
    (130, 1024, "bfloat16", "float32", 0, 2, "token", "float16", 0, 0.0),
    (9, 1025, "float32", "float32", 2, 1, "channel", "bfloat16", 3, 0.0),
    (777, 2883, "float32", "float16", 2, 2, "full", "float16", 0, 0.0),
    (17, 4096, "bfloat16", "bfloat16", 1, 1, "channel", "bfloat16", 8, 0.0),
    (4, 4104, "float16", "float16", 0, 2, None, "float32", 0, 1.0),
    (6, 8192, "float32", "bfloat16", 1, 2, "full", "float32", 0, 0.0),
    (3, 16384, "float32", "float32", 0, 1, "token", "float16", 0, 0.0),
    (3, 16385, "float32", "float32", 2, 2, "full", "float32", 0, 0.0),
    (2, 40000, "bfloat16", "float16", 1, 1, "channel", "bfloat16", 0, 0.0),
    (5000, 96, "bfloat16", "bfloat16", 0, 1, None, "bfloat16", 0, 0.0),     # more rows than a launch has workgroups
    (2500, 1536, "float32", "float32", 1, 1, "token", "float32", 0, 0.0),
    (512, 4095, "bfloat16", "bfloat16", 0, 1, None, "bfloat16", 1, 0.0), (513, 2049, "float16", "float16", 2, 1, "full", "float16", 0, 0.0),
]


@pytest.mark.parametrize("T,H,xt,ft,post,pre,gate,out,pad,w_add", CASES)
@pytest.mark.parametrize("i8", [False, True])
def test_norm(ctx, torch_dev, T, H, xt, ft, post, pre, gate, out, pad, w_add, i8):
    print("[case]", T, H, xt, ft, post, pre, gate, out, pad, i8, flush=True)
    torch = torch_dev
    rng = np.random.default_rng([T, H, post, pre])
    x = rows(torch, rng, T, H, xt, 3.0, pad)
    f = rows(torch, rng, T, H, ft, 0.5, pad) if ft else None
    shape = {None: None, "token": (T, 1), "channel": (1, H), "full": (T, H)}[gate]
    g = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(f.dtype).cuda() if shape else None
    vec = lambda: (1 - w_add + 0.2 * rng.standard_normal(H)).astype(np.float32)  # noqa: E731
    w, b, pw, pb = vec(), vec(), vec(), vec()
    if pre == 1:
        b = None
    d = lambda v: None if v is None else torch.from_numpy(v).cuda()  # noqa: E731
    alpha, eps = np.float32(0.7), 1e-5
    x_out, y = torch.zeros((T, H + pad), dtype=x.dtype, device="cuda")[:, :H], torch.zeros((T, H), dtype=getattr(torch, out), device="cuda")
    yq = torch.full((T, (H + 15) // 16 * 16), 99, dtype=torch.int8, device="cuda") if i8 else None
    ys = torch.zeros(T, device="cuda") if i8 else None
    torch.cuda.synchronize()
    ctx.norm(x, y=y, yq=yq, yscale=ys, kind=pre, w=d(w), b=d(b), eps=eps, w_add=w_add, x_out=x_out, branch=f, branch_kind=post if f is not None else 0,
             branch_w=d(pw) if f is not None and post else None, branch_b=d(pb) if f is not None and post == 2 else None, branch_eps=eps, gate=g,
             alpha=float(alpha))
    ctx.sync()
    v = host(x).astype(np.float64)
    if f is not None:
        n = I.normed(post, host(f), pw, pb if post == 2 else None, eps, w_add)
        v = v + np.float64(alpha) * (n if g is None else n * host(g))
    near(x_out, v, "x_out") if f is not None else None
    kept = host(x_out)                            # the row as stored is what the next norm reads
    if f is None:
        assert np.array_equal(kept, host(x))
    want = I.normed(pre, kept, w, b, eps, w_add)
    near(y, want, "y")
    if i8:
        q, s = I.quantize(want.astype(np.float32))
        assert np.array_equal(ys.cpu().numpy().view(np.uint32), s.view(np.uint32))
        assert np.array_equal(yq[:, :H].cpu().numpy(), q) and not yq[:, H:].any()


def test_in_place_and_single_outputs(ctx, torch_dev):
    import beglin_amd as B
    torch = torch_dev
    for T, H in ((3, 200), (2, 5000), (2, 17000)):
        rng = np.random.default_rng(H)
        x, f = rows(torch, rng, T, H, "float32"), rows(torch, rng, T, H, "float32")
        keep, y = x.clone(), torch.empty_like(x)
        torch.cuda.synchronize()
        ctx.norm(x, branch=f, x_out=x, y=y, kind=B.NORM_RMS)                    # the residual updated in place
        ctx.sync()
        v = (host(keep).astype(np.float64) + host(f)).astype(np.float32)
        assert np.array_equal(host(x), v)
        near(y, I.normed(1, v), "y")
        ctx.norm(x, branch=f, x_out=x, kind=B.NORM_NONE)                        # the last block: the add alone
        ctx.sync()
        v = (v.astype(np.float64) + host(f)).astype(np.float32)
        assert np.array_equal(host(x), v)
        ctx.norm(x, branch=f, y=y)                                              # no residual kept
        ctx.sync()
        near(y, I.normed(1, (v.astype(np.float64) + host(f)).astype(np.float32)), "y")
        assert np.array_equal(host(x), v)


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("T,H", [(3, 5), (2, 17000), (2, 33333)])
def test_16_bit_residual_rows_are_read_back(ctx, torch_dev, kind, T, H):
    """Rows that the kernel reads again for each pass (wider than 16384, narrower than 8): the new residual row is stored in 16
    bits and the norm, whose RMS waits at no barrier between the two, reads it back; beside x and in its place."""
    import beglin_amd as B
    torch = torch_dev
    rng = np.random.default_rng([T, H])
    x, f = rows(torch, rng, T, H, kind, 3.0), rows(torch, rng, T, H, kind, 0.5)
    v = (host(x).astype(np.float64) + host(f)).astype(np.float32)
    v = host(torch.from_numpy(v).to(x.dtype))               # the residual row as stored
    for pre in (B.NORM_RMS, B.NORM_NONE, B.NORM_LAYER):
        for src, place in ((x, torch.zeros_like(x)), (xc := x.clone(), xc)):
            y, yq, ys = torch.empty((T, H), device="cuda"), torch.zeros((T, (H + 15) // 16 * 16), dtype=torch.int8, device="cuda"), torch.empty(T, device="cuda")
            torch.cuda.synchronize()
            ctx.norm(src, branch=f, x_out=place, y=y, yq=yq, yscale=ys, kind=pre)
            ctx.sync()
            assert np.array_equal(host(place), v)
            want = I.normed(pre, v)
            near(y, want, "y")
            q, s = I.quantize(want.astype(np.float32))
            assert np.array_equal(yq[:, :H].cpu().numpy(), q) and np.array_equal(ys.cpu().numpy(), s)


@pytest.mark.parametrize("H", [48, 1536, 4096, 14336, 20000, 131056])
def test_quantizer_is_the_norm_of_kind_none(ctx, torch_dev, H):
    import beglin_amd as B
    torch = torch_dev
    rng = np.random.default_rng(H)
    x = rng.standard_normal((5, H)).astype(np.float32)
    x[1], x[2, 3], x[3, 4] = 0, np.nan, -np.inf
    xd = torch.from_numpy(x).cuda()
    out = [(torch.empty((5, H), dtype=torch.int8, device="cuda"), torch.empty(5, device="cuda")) for _ in range(2)]
    torch.cuda.synchronize()
    ctx.quant_act_i8(xd, H, *out[0])
    ctx.norm(xd, yq=out[1][0], yscale=out[1][1], kind=B.NORM_NONE)
    ctx.sync()
    q, s = I.quantize(x)
    for gq, gs in out:
        assert np.array_equal(gq.cpu().numpy(), q)
        gs = gs.cpu().numpy()
        assert np.array_equal(np.isnan(gs), np.isnan(s)) and np.array_equal(gs[~np.isnan(s)], s[~np.isnan(s)])


def test_non_finite_and_extreme_rows(ctx, torch_dev):
    """A row with NaN or an infinity gives NaN (as the formula does) and leaves the others alone; rows of 1e30 and 1e-30 keep
    their digits (the squares pass fp32's range), a row of zeros gives zeros."""
    import beglin_amd as B
    torch = torch_dev
    for H in (100, 3000, 20000):
        rng = np.random.default_rng(H)
        x = rng.standard_normal((6, H)).astype(np.float32)
        x[0] *= np.float32(1e30)
        x[1] *= np.float32(1e-30)
        x[2] = 0
        x[3, H // 2], x[4, 1] = np.nan, np.inf
        xd, y = torch.from_numpy(x).cuda(), torch.empty((6, H), device="cuda")
        yq, ys = torch.empty((6, (H + 15) // 16 * 16), dtype=torch.int8, device="cuda"), torch.empty(6, device="cuda")
        torch.cuda.synchronize()
        ctx.norm(xd, y=y, yq=yq, yscale=ys, kind=B.NORM_RMS, eps=0.0 if H == 100 else 1e-30)
        ctx.sync()
        got, s = y.cpu().numpy(), ys.cpu().numpy()
        eps = np.float64(np.float32(0.0 if H == 100 else 1e-30))
        want = x.astype(np.float64)
        with np.errstate(invalid="ignore"):
            want = want / np.sqrt((want * want).mean(-1, keepdims=True) + eps)
        for r in (0, 1, 5) if H == 100 else (0, 1, 2, 5):
            assert np.allclose(got[r], want[r], rtol=2.0 ** -23, atol=0), r
        assert np.isnan(got[3]).all() and np.isnan(s[3])
        assert np.isnan(got[4][1]) and not np.isfinite(s[4])
        assert not yq[3].any() and not yq[4].any()


def test_rows_past_4_gib(ctx, torch_dev):
    torch = torch_dev
    T, H = 140000, 16384
    x = torch.zeros((T, H), dtype=torch.bfloat16, device="cuda")
    some = torch.tensor([0, 1, 65537, 131071, 131072, T - 1])
    part = torch.from_numpy(np.random.default_rng(2).standard_normal((len(some), H)).astype(np.float32)).bfloat16()
    x[some.cuda()] = part.cuda()
    y, yq, ys = torch.empty_like(x), torch.empty((T, H), dtype=torch.int8, device="cuda"), torch.empty(T, device="cuda")
    torch.cuda.synchronize()
    ctx.norm(x, y=y, yq=yq, yscale=ys)
    ctx.sync()
    want = I.normed(1, host(part))
    near(y[some.cuda()], want, "y")
    q, s = I.quantize(want.astype(np.float32))
    assert np.array_equal(yq[some.cuda()].cpu().numpy(), q) and np.array_equal(ys[some.cuda()].cpu().numpy(), s)
    assert int((y != 0).any(1).sum()) == len(some) == int((yq != 0).any(1).sum())


def test_more_rows_than_a_launch_takes(ctx, torch_dev):
    torch = torch_dev
    T, H = (1 << 22) + 5, 8
    gen = torch.Generator(device="cuda").manual_seed(4)
    rand = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    x, f, g = rand(T, H), rand(T, H).half(), rand(T, 1).half()
    y, xo, yq, ys = torch.empty_like(x), torch.empty_like(x), torch.zeros((T, 16), dtype=torch.int8, device="cuda"), torch.empty(T, device="cuda")
    torch.cuda.synchronize()
    ctx.norm(x, y=y, yq=yq, yscale=ys, x_out=xo, branch=f, gate=g)
    ctx.sync()
    v = (x.double() + f.double() * g.double()).float()
    assert torch.equal(xo, v)
    n = v.double() / (v.double().square().mean(-1, keepdim=True) + float(np.float32(1e-6))).sqrt()
    assert ((y.double() - n).abs() <= n.abs() * (2.0 ** -24 * (1 + 1e-6)) + 1e-45).all()
    # (a tensor of 127s: torch multiplies by 1 / 127, rounded, where the divisor is a Python number)
    assert torch.equal(ys, y.abs().amax(-1) / torch.full_like(ys, 127.0))
    # half a code, and up to 127 codes times the roundings of the scale, its inverse, the two products and the difference
    assert ((yq[:, :H].float() * ys[:, None] - y).abs() <= ys[:, None] * (0.5 + 127 * 5 * 2.0 ** -24)).all()
