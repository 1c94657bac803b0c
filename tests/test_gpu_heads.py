"""bgl_heads_dev, bgl_kv_append_dev and bgl_kv_read_dev against the formulas in 64 bits.

A head's values for an fp32 output are computed in double and rounded to fp32, so a value may be off by half a step, 2^-24 relative; a
difference of two products that nearly cancel adds what a double's rounding (2^-53 of the products, far below 1e-13 of the
head's largest value) leaves.  For a 16-bit output fp32 arithmetic may stand in: a sum of squares in at most 8 + 6 additions,
halved by the root, with the division, root, products and the rotation's two roundings, (14 / 2 + 1 + 1 + 1 + 3 + 2) 2^-24 < 2^-20 of
the two products that are added, at most twice the largest value of the head; and half a step of the type, 2^-11 or 2^-8.  The cache's values
follow from the fp32 rows by single operations, so they are equal; where the rows pass through a norm or a rotation, a
value within 1e-10 of a border between two fp32 values may fall to either side, and with it one code to the next: such
codes are counted, and at most one in 10^5 may differ, by one step of its group."""
import numpy as np
import pytest

import kv_forms as F

pytestmark = pytest.mark.gpu
KINDS = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


@pytest.fixture(scope="module")
def torch_dev():
    import torch
    assert torch.cuda.is_available(), "gpu tests need a GPU"
    return torch


@pytest.fixture(scope="module")
def ctx(torch_dev):
    import beglin_amd
    st = torch_dev.cuda.Stream()                                                   # torch's work and the library's in one order
    c = beglin_amd.Context(0, st.cuda_stream)
    with torch_dev.cuda.stream(st):
        yield c
    c.sync()
    c.close()


def host(t):
    return t.float().cpu().numpy()


def near(got, want, name):
    kind = str(got.dtype).split(".")[1]
    rel = F.HALF["float32"] + (F.HALF[kind] if kind != "float32" else 0)
    g = host(got).astype(np.float64)
    sums = 1e-13 if kind == "float32" else 2 * 2.0 ** -20
    off = np.abs(g - want) - (rel * (1 + 1e-6) * np.abs(want) + F.LEAST[kind] + sums * np.abs(want).max(-1, keepdims=True))
    assert np.isfinite(g).all() and off.max() <= 0, (name, off.max(), np.argwhere(off > 0)[:4])


def rows(torch, rng, T, n, D, kind, layout="dense", scale=1.0):
    """[T][n][D] heads: dense, as a part of wider rows, with heads outermost, or off every alignment."""
    x = torch.from_numpy((rng.standard_normal((T, n, D)) * scale).astype(np.float32)).to(getattr(torch, KINDS[kind])).cuda()
    if layout == "dense":
        return x
    if layout == "part":
        wide = torch.zeros((T, n + 3, D), dtype=x.dtype, device="cuda")
        wide[:, 1:n + 1] = x
        return wide[:, 1:n + 1]
    if layout == "heads":
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros((T, n * (D + 1) + 1), dtype=x.dtype, device="cuda")         # "odd"
    view = wide[:, 1:].unflatten(1, (n, D + 1))[:, :, :D]
    view.copy_(x)
    return view


def rope_table(rng, n, rot):
    a = np.arange(n)[:, None] * 10000.0 ** (-np.arange(0, rot, 2) / rot)
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)


HEADS = [  # T, nq, nk, D, type, out, norm, style, rot, layout, w, w_add
    (1, 1, 1, 8, "f32", "f32", 1, 2, 8, "dense", True, 0.0),
    (1, 12, 2, 128, "f32", "f32", 0, 1, 128, "dense", False, 0.0),
    (3, 5, 1, 64, "f16", "bf16", 1, 1, 32, "part", True, 1.0),
    (2, 3, 3, 72, "bf16", "f32", 2, 2, 64, "heads", True, 0.0),
    (7, 6, 2, 96, "f16", "f16", 2, 2, 64, "odd", True, 0.0),
    (33, 40, 8, 128, "bf16", "bf16", 1, 1, 128, "part", True, 0.0),
    (257, 5, 5, 192, "f32", "f16", 1, 2, 192, "heads", False, 0.0),
    (65, 7, 1, 256, "bf16", "bf16", 2, 1, 256, "odd", True, 1.0),
    (19, 2, 2, 264, "f32", "f32", 1, 1, 16, "dense", True, 0.0),
    (5, 3, 2, 512, "f16", "f32", 1, 1, 512, "part", True, 0.0),
    (1031, 17, 3, 40, "f32", "f32", 0, 0, 0, "dense", False, 0.0),
    (1500, 33, 9, 80, "bf16", "f16", 1, 0, 0, "part", True, 0.0),
]


@pytest.mark.parametrize("case", HEADS, ids=["-".join(map(str, c)) for c in HEADS])
def test_heads(torch_dev, ctx, case):
    torch, (T, nq, nk, D, kind, out, norm, style, rot, layout, weights, w_add) = torch_dev, case
    rng = np.random.default_rng(T * 1000 + D)
    q, k = rows(torch, rng, T, nq, D, kind, layout, 3.0), rows(torch, rng, T, nk, D, kind, layout, 0.1)
    w = [(1 + 0.2 * rng.standard_normal(D)).astype(np.float32) if weights else None for _ in range(2)]
    wd = [None if x is None else torch.from_numpy(x).cuda() for x in w]
    n_pos = 50
    rope, pos = (rope_table(rng, n_pos, rot), rng.integers(0, n_pos, T).astype(np.int32)) if style else (None, None)
    if style and T > 6:
        pos[2], pos[5] = -1, n_pos                                                  # left alone
    kind_out = getattr(torch, KINDS[out])
    yq, yk = (torch.full_like(x, 7.0, dtype=kind_out) for x in (q, k))
    ctx.heads(q, k, yq, yk, norm=norm, q_w=wd[0], k_w=wd[1], eps=1e-5, w_add=w_add, rope=torch.from_numpy(rope).cuda() if style else None,
              pos=torch.from_numpy(pos).cuda() if style else None, rot=style)
    torch.cuda.synchronize()
    live = np.ones(T, bool) if not style else (pos >= 0) & (pos < n_pos)
    for x, y, wt, name in ((q, yq, w[0], "q"), (k, yk, w[1], "k")):
        want = F.heads(host(x), norm, wt, 1e-5, w_add, rope, pos, rot, style)
        near(y[torch.from_numpy(live).cuda()], want[live], name)
        assert (host(y)[~live] == 7.0).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("style", [1, 2])
def test_heads_in_place_and_one_of_two(torch_dev, ctx, kind, style):
    torch = torch_dev
    rng = np.random.default_rng(5)
    T, D = 37, 128
    q, k = rows(torch, rng, T, 6, D, kind, "part"), rows(torch, rng, T, 2, D, kind, "heads")
    rope, pos = rope_table(rng, 64, D), rng.integers(0, 64, T).astype(np.int32)
    how = dict(norm=1, rope=torch.from_numpy(rope).cuda(), pos=torch.from_numpy(pos).cuda(), rot=style)
    a, b, c, d = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q), torch.empty_like(k)
    ctx.heads(q, k, a, b, **how)
    ctx.heads(q, None, c, None, **how)
    ctx.heads(None, k, None, d, **how)
    ctx.heads(q, k, q, k, **how)
    torch.cuda.synchronize()
    for x, y in ((a, c), (b, d), (a, q), (b, k)):
        assert torch.equal(x, y)


def test_heads_rows_past_4_gib(torch_dev, ctx):
    """Tokens whose rows lie further than 2^32 bytes behind the first."""
    torch = torch_dev
    wide = torch.zeros((3, 3 << 29), dtype=torch.bfloat16, device="cuda")          # 3 GiB a row
    q = wide[:, 1000:1000 + 4 * 64].unflatten(1, (4, 64))
    x = torch.randn((3, 4, 64), device="cuda").bfloat16()
    q.copy_(x)
    a, b = torch.empty_like(x), torch.empty_like(x)
    ctx.heads(q, None, a, None, norm=1)
    ctx.heads(x, None, b, None, norm=1)
    ctx.heads(x, None, q, None, norm=1)
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.equal(q.contiguous(), b)
    assert int((wide[2].view(torch.int16) != 0).sum()) <= 256
    del wide, q
    torch.cuda.empty_cache()


def test_heads_of_extreme_rows(torch_dev, ctx):
    """All zeros, the largest and the smallest values: the norm of what a double holds."""
    torch = torch_dev
    x = torch.zeros((4, 2, 64), device="cuda")
    x[1] = 3e38
    x[2] = 1e-40
    x[3, 0, 5] = float("nan")
    y = torch.empty_like(x)
    ctx.heads(x, None, y, None, norm=1, eps=0.0)
    torch.cuda.synchronize()
    y = host(y)
    assert np.isnan(y[0]).all() and np.isnan(y[3, 0]).all() and np.isnan(y[3, 1]).all()
    assert np.allclose(y[1], 1, rtol=1e-7) and np.allclose(y[2], 1, rtol=1e-7)
    ctx.heads(x, None, torch.empty_like(x), None, norm=2, eps=1e-6)


def test_heads_of_extreme_16_bit_rows(torch_dev, ctx):
    """Rows whose squares leave fp32's range, beside ones that do not, through fp32 arithmetic."""
    torch = torch_dev
    rng = np.random.default_rng(2)
    x = rng.standard_normal((9, 3, 128)).astype(np.float32)
    x[1] *= 1e38
    x[2, 1] *= 1e20
    x[3] *= 1e-30
    x[4] = 0
    x[5, 0, 7] = np.inf
    x[6, 2, 100] = np.nan
    x[7] = 3e38
    q = torch.from_numpy(x).cuda().bfloat16()
    q[8] = float("-inf")
    rope, pos = rope_table(rng, 16, 128), np.arange(9, dtype=np.int32)
    y = torch.empty_like(q)
    w = (1 + 0.1 * rng.standard_normal(128)).astype(np.float32)
    ctx.heads(q, None, y, None, norm=1, q_w=torch.from_numpy(w).cuda(), eps=1e-6, rope=torch.from_numpy(rope).cuda(), pos=torch.from_numpy(pos).cuda())
    torch.cuda.synchronize()
    fine = np.isfinite(host(q)).all(-1)
    with np.errstate(invalid="ignore"):
        want = F.heads(host(q), 1, w, 1e-6, 0.0, rope, pos, 128, 1)
    assert not np.isfinite(host(y)[~fine]).all(-1).any()
    near(y[torch.from_numpy(fine).cuda()], want[fine], "finite rows")


def test_more_tokens_than_a_launch_takes(torch_dev, ctx):
    """2^20 tokens and some: launches of one call, and their slots and positions."""
    torch = torch_dev
    T, D, page, n = (1 << 20) + 37, 64, 256, 70
    gen = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn((T, 1, D), generator=gen, device="cuda").half() for _ in range(2))
    rope = torch.from_numpy(rope_table(np.random.default_rng(0), 512, D)).cuda()
    pos = (torch.arange(T, device="cuda") % 512).int()
    pages = T // page + 2
    slots = (torch.arange(T, device="cuda") + 3).int()
    whole, last = cache_of(torch, pages, page, 1, D), cache_of(torch, pages, page, 1, D)
    q, q2 = torch.empty_like(k), torch.empty_like(k)
    ctx.kv_append(whole, slots, k, v, q=k, q_out=q, norm=1, rope=rope, pos=pos)
    ctx.kv_append(last, slots[-n:], k[-n:], v[-n:], q=k[-n:], q_out=q2[-n:], norm=1, rope=rope, pos=pos[-n:])
    got = [torch.empty((T, 1, D), device="cuda") for _ in range(2)]
    ctx.kv_read(whole, slots, *got)
    few = [torch.empty((n, 1, D), device="cuda") for _ in range(2)]
    ctx.kv_read(last, slots[-n:], *few)
    ctx.heads(k, None, q2, None, norm=1, rope=rope, pos=pos)
    torch.cuda.synchronize()
    assert torch.equal(q, q2)
    for a, b in zip(got, few):
        assert torch.equal(a[-n:], b)
    assert torch.isfinite(got[0]).all() and torch.isfinite(got[1]).all()
    for at in (0, 1 << 19, (1 << 20) - 1, 1 << 20):
        assert np.array_equal(got[1][at].half().cpu().numpy(), F.kept(host(v[at])))


def cache_of(torch, pages, page, heads, D, fill=0xA5):
    import beglin_amd
    c = beglin_amd.KVCache(pages, page, heads, D)
    c.data.fill_(fill)
    return c


APPEND = [  # T, nq, nk, D, type, q out, norm, style, page, layout, first place
    (1, 0, 1, 64, "f32", "f32", 0, 0, 16, "dense", 0),
    (1, 4, 2, 128, "bf16", "bf16", 1, 1, 32, "part", 31),
    (8, 32, 8, 128, "bf16", "bf16", 1, 1, 64, "part", 3),
    (17, 6, 3, 96, "f16", "f32", 2, 2, 48, "odd", 5),
    (64, 5, 5, 64, "f32", "f16", 1, 2, 16, "heads", 0),
    (130, 2, 2, 192, "bf16", "bf16", 0, 1, 64, "dense", 2),
    (333, 8, 1, 256, "f16", "f16", 1, 1, 16, "odd", 9),
    (1001, 10, 5, 64, "f32", "f16", 0, 0, 256, "part", 1),
    (1200, 0, 4, 128, "f32", "f32", 0, 0, 128, "heads", 4),
    (600, 32, 2, 128, "bf16", "bf16", 1, 1, 64, "part", 7),                        # queries enough for a launch of their own
    (1500, 12, 3, 64, "f16", "bf16", 0, 2, 16, "odd", 1),
]


@pytest.mark.parametrize("case", APPEND, ids=["-".join(map(str, c)) for c in APPEND])
def test_append_and_read(torch_dev, ctx, case):
    torch, (T, nq, nk, D, kind, out, norm, style, page, layout, first) = torch_dev, case
    rng = np.random.default_rng(T + D)
    k, v = rows(torch, rng, T, nk, D, kind, layout, 2.0), rows(torch, rng, T, nk, D, kind, layout)
    q = rows(torch, rng, T, nq, D, kind, layout) if nq else None
    w = [(1 + 0.2 * rng.standard_normal(D)).astype(np.float32) for _ in range(2)]
    rope, pos = (rope_table(rng, 2000, D), (np.arange(T) + 7).astype(np.int32)) if style else (None, None)
    pages = (T + first + page - 1) // page + 2
    order = rng.permutation(pages)
    at = np.arange(T) + first
    slots = (order[at // page] * page + at % page).astype(np.int32)
    if T > 8:
        slots[4], slots[7], slots[T - 1] = -1, pages * page, -2 ** 31              # nowhere
    cache = cache_of(torch, pages, page, nk, D)
    before = cache.data.clone()
    yq = torch.empty((T, nq, D), dtype=getattr(torch, KINDS[out]), device="cuda") if nq else None
    sd = torch.from_numpy(slots).cuda()
    ctx.kv_append(cache, sd, k, v, q=q, q_out=yq, norm=norm, q_w=torch.from_numpy(w[0]).cuda(), k_w=torch.from_numpy(w[1]).cuda(), eps=1e-6,
                  rope=torch.from_numpy(rope).cuda() if style else None, pos=torch.from_numpy(pos).cuda() if style else None, rot=style)
    got_k, got_v = (torch.full((T, nk, D), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    ctx.kv_read(cache, sd, got_k, got_v)
    torch.cuda.synchronize()
    live = (slots >= 0) & (slots < pages * page)
    if nq:
        near(yq, F.heads(host(q), norm, w[0], 1e-6, 0.0, rope, pos, D, style), "q")
    want_k = F.kept(F.heads(host(k), norm, w[1], 1e-6, 0.0, rope, pos, D, style).astype(np.float32))[live]
    want_v = F.kept(host(v))[live]
    gk, gv = got_k.cpu().numpy(), got_v.cpu().numpy()
    assert (gk[~live] == 7).all() and (gv[~live] == 7).all()
    assert np.array_equal(gv[live], want_v)
    differ = gk[live] != want_k
    assert differ.mean() <= (1e-5 if norm or style else 0), differ.mean()
    # the records themselves, and that nothing else was written
    rec = cache.data.cpu().numpy().reshape(pages, nk, page // 16, 20 * D)
    old = before.cpu().numpy().reshape(rec.shape)
    used = set()
    for i in np.flatnonzero(live)[:: max(1, T // 5)]:
        pg, place = divmod(int(slots[i]), page)
        h = int(rng.integers(nk))
        rk, rv = F.record_values(rec[pg, h, place // 16], D)
        assert np.array_equal(rk[place % 16], gk[i, h]) and np.array_equal(rv[place % 16], gv[i, h])
    for s in slots[live]:
        used.add((int(s) // page, int(s) % page // 16))
    for pg in range(pages):
        for t in range(page // 16):
            if (pg, t) not in used:
                assert np.array_equal(rec[pg, :, t], old[pg, :, t])
    # tokens without a place, inside records that others were written to
    mark = [pg * page + t * 16 + i for pg, t in list(used)[:3] for i in range(16)]
    free = np.array([m for m in mark if m not in set(slots[live].tolist())][:8], np.int32)
    if len(free):
        for m in free:
            pg, place = divmod(int(m), page)
            a, b = F.record_values(rec[pg, 0, place // 16], D), F.record_values(old[pg, 0, place // 16], D)
            for x, y in zip(a, b):
                assert np.array_equal(x[place % 16].view(np.uint16), y[place % 16].view(np.uint16))


@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
def test_read_types_and_one_of_two(torch_dev, ctx, type_):
    torch = torch_dev
    rng = np.random.default_rng(3)
    T, nk, D = 21, 3, 96
    k, v = rows(torch, rng, T, nk, D, "f32"), rows(torch, rng, T, nk, D, "f32")
    cache = cache_of(torch, 4, 16, nk, D)
    slots = torch.arange(T, dtype=torch.int32, device="cuda") + 3
    ctx.kv_append(cache, slots, k, v)
    kind = getattr(torch, KINDS[type_])
    gk, gv, wide = (torch.zeros((T, nk, D), dtype=kind, device="cuda") for _ in range(3))
    ctx.kv_read(cache, slots, gk, None)
    ctx.kv_read(cache, slots, None, gv)
    part = rows(torch, rng, T, nk, D, type_, "heads")
    ctx.kv_read(cache, slots, part, wide)
    torch.cuda.synchronize()
    assert torch.equal(gk, torch.from_numpy(F.kept(host(k))).cuda().float().to(kind)) and torch.equal(part, gk)
    assert torch.equal(gv, torch.from_numpy(F.kept(host(v))).cuda().float().to(kind)) and torch.equal(wide, gv)


def test_append_of_odd_groups(torch_dev, ctx):
    """Groups of one value, of steps below fp16's smallest, past +-32768, with a NaN or an infinity."""
    torch = torch_dev
    D = 64
    x = np.random.default_rng(1).standard_normal((12, 1, D)).astype(np.float32)
    x[0] = 0.0
    x[1] = -1.0001
    x[2] = 3.0 + 1e-7 * x[2]
    x[3] *= 1e30
    x[4] *= 1e-20
    x[5, 0, 3] = np.nan
    x[6, 0, 40] = np.inf
    x[7, 0, :32] = -np.inf
    x[8, 0, 0], x[8, 0, 1] = 65504.0, -65504.0
    x[9] = 40000.0
    x[10, 0, 31] = 1000.0
    x[11] = -0.0
    cache = cache_of(torch, 1, 16, 1, D)
    slots = torch.arange(12, dtype=torch.int32, device="cuda")
    xd = torch.from_numpy(x).cuda()
    k, v = torch.zeros((12, 1, D), dtype=torch.float16, device="cuda"), torch.zeros((12, 1, D), dtype=torch.float16, device="cuda")
    ctx.kv_append(cache, slots, xd, torch.from_numpy(x).cuda())
    ctx.kv_read(cache, slots, k, v)
    torch.cuda.synchronize()
    want = F.kept(x)
    for got in (k, v):
        assert np.array_equal(got.cpu().numpy(), want, equal_nan=True)
    assert np.isnan(want[5, 0, :32]).all() and np.isfinite(want[5, 0, 32:]).all()


def test_pack_is_what_append_writes(torch_dev, ctx):
    torch = torch_dev
    rng = np.random.default_rng(8)
    for D in (64, 96, 128, 192, 256):
        k, v = (rng.standard_normal((16, 1, D)).astype(np.float32) for _ in range(2))
        cache = cache_of(torch, 1, 16, 1, D)
        ctx.kv_append(cache, torch.arange(16, dtype=torch.int32, device="cuda"), torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
        torch.cuda.synchronize()
        assert np.array_equal(cache.data.cpu().numpy(), F.pack(k.reshape(1, 16, D), v.reshape(1, 16, D))[0])


def test_append_is_captured_and_replayed(torch_dev):
    """A graph that appends each step's tokens where its slots say, beside eager calls of the same context."""
    import beglin_amd as B
    torch = torch_dev
    rng = np.random.default_rng(11)
    st = torch.cuda.Stream()
    c = B.Context(0, st.cuda_stream)
    T, nq, nk, D, page = 6, 8, 2, 128, 16
    cache, other = cache_of(torch, 8, page, nk, D), cache_of(torch, 8, page, nk, D)
    q, k, v = (rows(torch, rng, T, n, D, "bf16") for n in (nq, nk, nk))
    rope = torch.from_numpy(rope_table(rng, 256, D)).cuda()
    slots, pos = torch.zeros(T, dtype=torch.int32, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda")
    yq, eq = torch.empty_like(q), torch.empty_like(q)
    call = lambda kv, out: c.kv_append(kv, slots, k, v, q=q, q_out=out, norm=1, rope=rope, pos=pos)  # noqa: E731
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            call(cache, yq)
        for step in range(4):
            slots.copy_(torch.arange(T, dtype=torch.int32) * page + step)
            pos.fill_(20 * step)
            k.copy_(torch.randn(k.shape))
            v.copy_(torch.randn(v.shape))
            g.replay()
            call(other, eq)
            st.synchronize()
            assert torch.equal(yq, eq) and torch.equal(cache.data, other.data), step
    c.close()
