"""bgl_attn_dev against attention in 64 bits over the values that the cache stands for (kv_forms.attention_near has the tolerances)."""
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


class Batch:
    """Sequences of (rows, keys) over a cache whose other places, and whose table's other entries, hold anything."""

    def __init__(self, torch, ctx, seqs, nq, nk, D, kind, page, seed=0, poison=(), gone=(), scale_q=1.0, scale_k=1.0, layout="dense"):
        import beglin_amd
        rng = np.random.default_rng(seed)
        self.torch, self.seqs, self.nq, self.nk, self.D, self.page = torch, seqs, nq, nk, D, page
        need = [(n + page - 1) // page for _, n in seqs]
        pages = sum(need) + 3
        self.cache = beglin_amd.KVCache(pages, page, nk, D)
        self.cache.data.fill_(0xFF)                                                # NaN everywhere
        order = rng.permutation(pages).astype(np.int32)
        wide = max(need + [1]) + 1
        table = rng.choice(np.array([-1, 2 ** 31 - 1, -2 ** 31, pages, pages + 7, order[-1]]), (len(seqs), wide)).astype(np.int32)
        self.k, self.v, at = [], [], 0
        for s, (_, n) in enumerate(seqs):
            table[s, :need[s]] = order[at:at + need[s]]
            at += need[s]
            if not n:
                self.k.append(np.zeros((0, nk, D))), self.v.append(np.zeros((0, nk, D)))
                continue
            k = (rng.standard_normal((n, nk, D)) * scale_k).astype(np.float32)
            k[:, :, :3] *= 5
            v = (rng.standard_normal((n, nk, D)) + 0.3).astype(np.float32)
            for (t, j, h, d, which) in poison:
                if t == s:
                    (k if which == "k" else v)[j, h, d] = np.nan if d % 2 else np.inf
            j = np.arange(n)
            slots = torch.from_numpy((table[s, j // page] * page + j % page).astype(np.int32)).cuda()
            ctx.kv_append(self.cache, slots, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
            gk, gv = (torch.empty((n, nk, D), dtype=torch.float16, device="cuda") for _ in range(2))
            ctx.kv_read(self.cache, slots, gk, gv)
            torch.cuda.synchronize()
            self.k.append(gk.cpu().numpy()), self.v.append(gv.cpu().numpy())
        self.gone = gone                                                           # (sequence, page) whose entry names no page
        for s, p in gone:
            table[s, p] = -1 if p % 2 else pages
        self.start = np.concatenate([[0], np.cumsum([r for r, _ in seqs])]).astype(np.int32)
        self.T = int(self.start[-1])
        self.extra = 2                                                             # rows behind the last sequence
        q = (rng.standard_normal((self.T + self.extra, nq, D)) * scale_q).astype(np.float32)
        dt = getattr(torch, KINDS[kind])
        q = torch.from_numpy(q).to(dt).cuda()
        if layout == "heads":
            q = q.transpose(0, 1).contiguous().transpose(0, 1)
        elif layout == "part":
            w = torch.zeros((q.shape[0], nq + 2 * nk, D), dtype=dt, device="cuda")
            w[:, :nq] = q
            q = w[:, :nq]
        elif layout == "odd":
            w = torch.zeros((q.shape[0], nq * (D + 1) + 1), dtype=dt, device="cuda")[:, 1:].unflatten(1, (nq, D + 1))[:, :, :D]
            w.copy_(q)
            q = w
        self.q = q
        self.out = torch.full_like(q, 7.0)
        self.sink = rng.standard_normal(nq).astype(np.float32) * 2
        dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
        self.start_d, self.lens_d, self.table_d = dev(self.start), dev(np.array([n for _, n in seqs], np.int32)), dev(table)

    def run(self, ctx, sink=False, **how):
        ctx.attention(self.cache, self.q, self.out, self.start_d, self.lens_d, self.table_d,
                      sink=self.torch.from_numpy(self.sink).cuda() if sink else None, **how)
        self.torch.cuda.synchronize()
        return host(self.out)

    def seen(self, s, causal, window):
        r, n = self.seqs[s]
        pos, key = np.arange(n - r, n)[:, None], np.arange(n)[None]
        see = (key <= pos) if causal else np.ones((r, n), bool)
        if window:
            see = see & (key > pos - window)
        for t, p in self.gone:
            if t == s:
                see = see & (key // self.page != p)
        return see

    def check(self, got, causal=True, window=0, sink=False, scale=None, only=None):
        D, q = self.D, host(self.q).astype(np.float64)
        kind = str(self.q.dtype).split(".")[1]
        scale = D ** -0.5 if scale is None else scale
        g = self.nq // self.nk
        for s, (r, n) in enumerate(self.seqs):
            if only is not None and s not in only:
                continue
            see = self.seen(s, causal, window)
            for h in range(self.nq):
                rows = slice(self.start[s], self.start[s] + r)
                F.attention_near(got[rows, h], q[rows, h], self.k[s][:, h // g], self.v[s][:, h // g], scale, see, self.sink[h] if sink else None, kind, (s, h))
        assert (got[self.T:] == 7).all(), "rows of no sequence"


DECODE = [  # sequences (rows, keys), nq, nk, D, type, page, layout
    ([(1, 1)], 1, 1, 64, "f32", 16, "dense"),
    ([(1, 2), (1, 0), (0, 5), (1, 16), (1, 17)], 2, 1, 128, "f16", 16, "dense"),
    ([(1, 31), (1, 32), (1, 33), (1, 127), (1, 128), (1, 129)], 12, 2, 128, "f32", 16, "part"),
    ([(1, 300)], 12, 2, 128, "bf16", 48, "heads"),
    ([(1, 700), (1, 3), (1, 1500)], 8, 8, 64, "bf16", 64, "odd"),
    ([(1, 257), (1, 96)], 16, 1, 96, "f16", 32, "odd"),
    ([(1, 513), (1, 65)], 6, 3, 96, "f32", 48, "part"),
    ([(1, 400)], 10, 2, 192, "bf16", 16, "heads"),
    ([(1, 333), (1, 40)], 3, 1, 192, "f32", 64, "dense"),
    ([(1, 640), (1, 100)], 16, 2, 256, "f16", 128, "dense"),
    ([(1, 200), (1, 90)], 4, 4, 256, "f32", 16, "odd"),
    ([(3, 200), (1, 77), (2, 2), (4, 500)], 8, 2, 128, "bf16", 32, "part"),
    ([(5, 100), (8, 8), (7, 300)], 8, 2, 64, "f32", 16, "dense"),                  # up to 32 rows of a head
    ([(3, 130), (2, 259)], 20, 2, 128, "f32", 32, "heads"),
    ([(5, 70)], 7, 1, 96, "f16", 16, "dense"),
    ([(3, 90), (9, 60)], 14, 2, 256, "bf16", 16, "dense"),                         # several blocks of rows
    ([(5, 3), (9, 4), (3, 1)], 4, 1, 64, "f16", 16, "dense"),                      # more rows than keys
    ([(1, 20000)], 4, 1, 128, "bf16", 128, "dense"),
    ([(1, 9000), (2, 1), (1, 3000)], 4, 2, 64, "f32", 16, "dense"),
    ([(1, 5000), (1, 4095), (1, 4097)], 4, 4, 64, "f16", 4096, "dense"),
    ([(1, 2500), (3, 1009)], 3, 1, 128, "bf16", 1008, "part"),
    ([(1, 50)], 70, 70, 64, "bf16", 16, "dense"),                                  # many heads
]


@pytest.mark.parametrize("case", DECODE, ids=[str(i) for i in range(len(DECODE))])
def test_few_rows(torch_dev, ctx, case):
    seqs, nq, nk, D, kind, page, layout = case
    b = Batch(torch_dev, ctx, seqs, nq, nk, D, kind, page, layout=layout)
    b.check(b.run(ctx))
    b.out.fill_(7.0)
    b.check(b.run(ctx, sink=True, causal=False, scale=0.3), causal=False, sink=True, scale=0.3)
    b.out.fill_(7.0)
    b.check(b.run(ctx, window=21, scale=-0.05, max_rows=1, max_len=1), window=21, scale=-0.05)
    b.out.fill_(7.0)
    b.check(b.run(ctx, window=200, sink=True, max_rows=1000, max_len=10 ** 6), window=200, sink=True)


PROMPTS = [  # sequences (rows, keys), nq, nk, D, type, page, layout
    ([(33, 33)], 1, 1, 64, "f32", 16, "dense"),
    ([(300, 300)], 4, 1, 128, "bf16", 32, "part"),
    ([(130, 700)], 6, 2, 128, "f32", 48, "heads"),
    ([(64, 1000), (1, 500), (70, 70), (0, 40), (2, 300)], 8, 2, 64, "f16", 16, "odd"),
    ([(40, 90), (257, 300)], 6, 6, 96, "f16", 32, "dense"),
    ([(100, 130)], 2, 1, 96, "f32", 16, "odd"),
    ([(77, 200), (5, 64), (129, 129)], 4, 2, 192, "bf16", 64, "part"),
    ([(90, 90)], 3, 1, 192, "f32", 16, "dense"),
    ([(50, 333), (1, 1)], 16, 2, 256, "bf16", 16, "dense"),
    ([(60, 61)], 2, 2, 256, "f32", 48, "heads"),
    ([(45, 12), (70, 65)], 2, 1, 128, "bf16", 16, "dense"),                        # more rows than keys
    ([(40, 6000)], 1, 1, 128, "f16", 128, "dense"),                                # few rows, many keys: in parts
    ([(200, 4000)], 4, 2, 64, "f32", 64, "dense"),
]


@pytest.mark.parametrize("case", PROMPTS, ids=[str(i) for i in range(len(PROMPTS))])
def test_many_rows(torch_dev, ctx, case):
    seqs, nq, nk, D, kind, page, layout = case
    b = Batch(torch_dev, ctx, seqs, nq, nk, D, kind, page, layout=layout)
    most, longest = max(r for r, _ in seqs), max(n for _, n in seqs)
    b.check(b.run(ctx))
    b.out.fill_(7.0)
    b.check(b.run(ctx, sink=True, causal=False, scale=0.3, max_rows=most, max_len=longest), causal=False, sink=True, scale=0.3)
    b.out.fill_(7.0)
    b.check(b.run(ctx, window=21, scale=-0.05, max_rows=33, max_len=1), window=21, scale=-0.05)
    b.out.fill_(7.0)
    b.check(b.run(ctx, window=100, sink=True, max_rows=40, max_len=10 ** 6), window=100, sink=True)
    b.out.fill_(7.0)
    b.check(b.run(ctx, max_rows=1, max_len=longest))
    b.out.fill_(7.0)
    b.check(b.run(ctx, max_len=10 ** 6))                                           # the largest blocks, their keys in many parts


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
def test_many_rows_of_many_heads(torch_dev, ctx, kind, D):
    """More blocks than CUs, so the largest ones, in one part."""
    b = Batch(torch_dev, ctx, [(70, 300), (60, 130), (40, 40), (5, 90), (110, 700), (35, 2000)], 90, 90, D, kind, 32)
    b.check(b.run(ctx))
    b.out.fill_(7.0)
    b.check(b.run(ctx, sink=True, window=77), sink=True, window=77)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("window", [0, 30])
def test_nan_and_pages_that_are_gone_among_many_rows(torch_dev, ctx, kind, D, window):
    last = D - 1
    poison = [(0, 95, 0, 3, "k"), (0, 80, 1, 40, "v"), (1, 60, 1, last, "v"), (1, 51, 0, 1, "v"), (2, 5, 0, last, "k"), (3, 2, 1, 2, "v"), (3, 17, 0, 33, "v")]
    b = Batch(torch_dev, ctx, [(40, 97), (34, 63), (1, 6), (36, 36), (50, 50)], 4, 2, D, kind, 16, poison=poison, gone=[(0, 2), (4, 0), (4, 2), (1, 3)])
    b.q[-4, 1, 5] = float("inf")
    b.q[-3, 0, 0] = float("nan")
    b.check(b.run(ctx, window=window), window=window)
    b.out.fill_(7.0)
    b.check(b.run(ctx, window=window, sink=True, max_rows=50, max_len=97), window=window, sink=True)
    b.out.fill_(7.0)
    b.check(b.run(ctx, window=window, max_rows=50, max_len=10 ** 6), window=window)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
def test_pages_that_are_gone(torch_dev, ctx, kind, D):
    """Table entries that name no page hide their keys; a row may be left without any."""
    b = Batch(torch_dev, ctx, [(2, 150), (1, 20), (1, 33)], 4, 2, D, kind, 16, gone=[(0, 0), (0, 1), (0, 5), (1, 0), (1, 1), (2, 2)])
    got = b.run(ctx)
    b.check(got)
    assert (got[2] == 0).all()
    b.out.fill_(7.0)
    b.check(b.run(ctx, sink=True, window=40), sink=True, window=40)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("window", [0, 9])
def test_nan_reaches_the_rows_that_see_it(torch_dev, ctx, kind, D, window):
    """NaN and infinities among keys (a row that sees one is NaN) and values (its 32 values are), on both sides of the rows' diagonal
    and of the window's edge."""
    last = D - 1
    poison = [(0, 95, 0, 3, "k"), (0, 93, 1, 40, "v"), (1, 60, 1, last, "v"), (1, 51, 0, 1, "v"), (2, 5, 0, last, "k"), (3, 2, 1, 2, "v")]
    b = Batch(torch_dev, ctx, [(6, 97), (8, 63), (1, 6), (4, 4), (2, 50)], 4, 2, D, kind, 16, poison=poison)
    b.q[-4, 1, 5] = float("inf")                                                   # a query as well (of the last sequence)
    b.q[-3, 0, 0] = float("nan")
    b.check(b.run(ctx, window=window), window=window)


def test_queries_of_any_size(torch_dev, ctx):
    """Rows whose values lie far apart or far from 1: a row is scaled by its largest value."""
    torch = torch_dev
    for kind, sizes in (("f32", (1e-30, 1e-3, 1.0, 50.0)), ("bf16", (1e-30, 1.0, 300.0)), ("f16", (1e-6, 1.0, 30.0))):
        b = Batch(torch, ctx, [(len(sizes), 70)], 2, 1, 128, kind, 16)
        for i, z in enumerate(sizes):
            b.q[i] *= z
        b.q[0, 0] = 0
        b.check(b.run(ctx))


def test_scores_far_apart(torch_dev, ctx):
    """Scores in the hundreds: one key takes all, in one part of the keys or another."""
    for kind in ("f32", "f16", "bf16"):
        b = Batch(torch_dev, ctx, [(1, 900), (2, 450)], 4, 1, 128, kind, 32, scale_q=8.0, scale_k=6.0)
        b.check(b.run(ctx))


def test_same_bits_every_time(torch_dev, ctx):
    torch = torch_dev
    for seqs in ([(1, n) for n in (4000, 17, 900, 2500, 1, 333)], [(40, 3000), (90, 200), (1, 50)]):
        b = Batch(torch, ctx, seqs, 8, 2, 128, "bf16", 64)
        first = b.run(ctx).copy()
        for _ in range(5):
            b.out.fill_(3.0)
            assert np.array_equal(b.run(ctx)[:b.T], first[:b.T])


def test_many_sequences(torch_dev, ctx):
    """More sequences than a workgroup has threads, some without rows or keys."""
    rng = np.random.default_rng(2)
    seqs = [(int(rng.integers(0, 3)), int(rng.integers(0, 70))) for _ in range(700)]
    seqs = [(min(r, max(n, 1)), n) for r, n in seqs]
    b = Batch(torch_dev, ctx, seqs[:300], 2, 1, 64, "f16", 16)
    b.check(b.run(ctx))
    b.out.fill_(7.0)
    b.check(b.run(ctx, window=5, sink=True), window=5, sink=True)


@pytest.mark.parametrize("case", [(30, 3000, 12, 1), (90, 900, 20, 1), (50, 2600, 40, 1), (25, 2000, 10, 4)], ids=str)
def test_lengths_far_apart(torch_dev, ctx, case):
    """Units for every workgroup several times over, and sequences of few of them between long ones."""
    count, longest, heads, most = case
    rng = np.random.default_rng(count)
    lens = np.exp(rng.uniform(0, np.log(longest), count)).astype(int)
    lens[::7] = longest
    seqs = [(int(rng.integers(0, most + 1)) if most > 1 else 1, int(n)) for n in lens]
    b = Batch(torch_dev, ctx, seqs, heads, heads, 64, "bf16", 32)
    b.check(b.run(ctx, max_rows=most))
    b.out.fill_(7.0)
    b.check(b.run(ctx, max_rows=most, max_len=longest, window=700), window=700)
    again = b.run(ctx, max_rows=most, max_len=longest, window=700)
    assert np.array_equal(again[:b.T], b.run(ctx, max_rows=most, max_len=longest, window=700)[:b.T])


def test_bad_starts_and_lengths_stay_in_bounds(torch_dev, ctx):
    """start and len are read on the device: rows outside [0, T) and keys outside the table do not exist."""
    torch = torch_dev
    b = Batch(torch, ctx, [(1, 40), (1, 50), (1, 30)], 2, 1, 64, "f32", 16)
    want = b.run(ctx).copy()
    b.lens_d[0] = -7
    b.lens_d[2] = 2 ** 31 - 1                                                      # its table's entries past the pages name none, or NaN
    b.start_d[0] = -2 ** 31
    b.start_d[3] = 2 ** 31 - 1
    b.out.fill_(7.0)
    got = b.run(ctx)
    assert np.array_equal(got[1], want[1])


@pytest.mark.parametrize("hint", [None, 1])
def test_starts_that_go_back_stay_in_bounds(torch_dev, ctx, hint):
    torch = torch_dev
    b = Batch(torch, ctx, [(9, 40), (5, 50), (20, 300)], 4, 1, 64, "f16", 16)
    b.start_d.copy_(torch.tensor([0, 30, 4, 34], dtype=torch.int32))
    got = b.run(ctx, max_rows=hint)
    assert (got[b.T:] == 7.0).all()
    b.start_d.copy_(torch.from_numpy(b.start))
    b.check(b.run(ctx, max_rows=hint))


@pytest.mark.parametrize("rows", [1, 40])
def test_sinks_without_end(torch_dev, ctx, rows):
    """exp(sink) of infinity leaves a row 0, of -infinity as it is without one, NaN makes NaN."""
    b = Batch(torch_dev, ctx, [(rows, 100), (rows, 3000), (rows, 0)], 4, 2, 64, "bf16", 16)
    want = b.run(ctx).copy()
    b.sink[:] = np.array([np.inf, -np.inf, 3e38, np.nan], np.float32)
    got = b.run(ctx, sink=True)[:b.T]
    assert (got[:, 0] == 0).all() and (got[:, 2] == 0).all()
    assert np.array_equal(got[:, 1], want[:b.T, 1])
    assert np.isnan(got[:2 * rows, 3]).all() and (got[2 * rows:, 3] == 0).all()      # a row without a key is 0 whatever the sink


def test_a_prompt_among_many_sequences(torch_dev, ctx):
    """More blocks of rows than a launch takes: a workgroup goes over several."""
    torch = torch_dev
    import beglin_amd
    nq, nk, D, page, n, S = 32, 8, 64, 64, 36000, 2001
    cache = beglin_amd.KVCache(n // page + 1, page, nk, D)
    gen = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn((n, nk, D), generator=gen, device="cuda") for _ in range(2))
    ctx.kv_append(cache, torch.arange(n, dtype=torch.int32, device="cuda"), k, v)
    q = torch.randn((n + S - 1, nq, D), generator=gen, device="cuda").half()
    pages = torch.arange(cache.pages, dtype=torch.int32, device="cuda")
    out, one = torch.full_like(q, 7.0), torch.full_like(q[:n], 7.0)
    start = torch.arange(S + 1, dtype=torch.int32, device="cuda")
    start[S] = n + S - 1
    lens = 1 + start[1:] % 16
    lens[S - 1] = n
    ctx.attention(cache, q, out, start, lens, pages[None].repeat(S, 1))
    ctx.attention(cache, q[S - 1:], one, torch.tensor([0, n], dtype=torch.int32, device="cuda"), lens[S - 1:].contiguous(), pages[None])
    few = torch.empty_like(q[:S - 1])
    ctx.attention(cache, q[:S - 1], few, start[:S].contiguous(), lens[:S - 1].contiguous(), pages[None, :1].repeat(S - 1, 1), max_rows=1)
    torch.cuda.synchronize()
    assert torch.equal(out[S - 1:], one)
    apart = np.abs(host(out[:S - 1]) - host(few)).max()
    assert apart <= 2 ** -9 * np.abs(host(v[:16])).max()                           # two results, each off by a rounding of weights and one of the output


def test_cache_past_4_gib(torch_dev, ctx):
    """Pages whose records lie further than 2^32 bytes behind the first, and q rows that do."""
    import beglin_amd
    torch = torch_dev
    page, nk, D = 256, 8, 128
    per = page // 16 * nk * 20 * D
    pages = (5 << 30) // per
    cache = beglin_amd.KVCache(pages, page, nk, D)
    small = beglin_amd.KVCache(3, page, nk, D)
    n = 600
    rng = np.random.default_rng(4)
    k, v = (torch.from_numpy(rng.standard_normal((n, nk, D)).astype(np.float32)).cuda() for _ in range(2))
    tables = []
    for c, ids in ((cache, [pages - 1, 3, pages - 2]), (small, [0, 1, 2])):
        ids = np.array(ids, np.int32)
        at = np.arange(n)
        slots = torch.from_numpy((ids[at // page].astype(np.int64) * page + at % page).astype(np.int32)).cuda()
        ctx.kv_append(c, slots, k, v)
        tables.append(torch.from_numpy(ids[None]).cuda())
        a, e = torch.empty((n, nk, D), device="cuda"), torch.empty((n, nk, D), device="cuda")
        ctx.kv_read(c, slots, a, e)
        torch.cuda.synchronize()
        assert np.array_equal(a.cpu().numpy(), F.kept(k.cpu().numpy()).astype(np.float32))
    q = torch.from_numpy(rng.standard_normal((2, 16, D)).astype(np.float32)).cuda()
    start, lens = torch.tensor([0, 2], dtype=torch.int32, device="cuda"), torch.tensor([n], dtype=torch.int32, device="cuda")
    outs = []
    for c, t in zip((cache, small), tables):
        out = torch.empty_like(q)
        ctx.attention(c, q, out, start, lens, t)
        outs.append(out)
    torch.cuda.synchronize()
    assert torch.equal(*outs)
    del cache
    torch.cuda.empty_cache()


def test_rows_of_queries_past_4_gib(torch_dev, ctx):
    torch = torch_dev
    b = Batch(torch, ctx, [(2, 200), (1, 70)], 4, 2, 64, "bf16", 16)
    want = b.run(ctx)[:3].copy()
    wide = torch.zeros((3, 3 << 29), dtype=torch.bfloat16, device="cuda")          # 3 GiB a row
    q, out = (wide[:, at:at + 256].unflatten(1, (4, 64)) for at in (1000, 2000))
    q.copy_(b.q[:3])
    ctx.attention(b.cache, q, out, b.start_d, b.lens_d, b.table_d)
    torch.cuda.synchronize()
    assert np.array_equal(host(out), want)
    ctx.attention(b.cache, q, out, torch.tensor([0, 3], dtype=torch.int32, device="cuda"), b.lens_d[:1], b.table_d[:1], max_rows=3)
    torch.cuda.synchronize()
    assert np.isfinite(host(out)).all()
    del wide, q, out
    torch.cuda.empty_cache()


def test_two_contexts_at_once(torch_dev, ctx):
    """Calls of two contexts on two streams, which nothing orders: each has scratch of its own."""
    import beglin_amd as B
    torch = torch_dev
    batches = [Batch(torch, ctx, seqs, 8, 2, 128, "bf16", 64, seed=i) for i, seqs in enumerate(([(1, 6000), (1, 300)], [(1, 5000), (2, 2500), (60, 2000)]))]
    want = [b.run(ctx)[:b.T].copy() for b in batches]
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [B.Context(0, s.cuda_stream) for s in streams]
    for _ in range(8):
        for b in batches:
            b.out.fill_(7.0)
        torch.cuda.synchronize()
        for _ in range(10):
            for c, b in zip(ctxs, batches):
                c.attention(b.cache, b.q, b.out, b.start_d, b.lens_d, b.table_d)
        torch.cuda.synchronize()
        for b, w in zip(batches, want):
            assert np.array_equal(host(b.out)[:b.T], w)
    for c in ctxs:
        c.close()


def test_captured_decode_steps(torch_dev):
    """append and attention of a step as one graph, replayed as the sequences grow, beside eager calls of the same context on other buffers."""
    import beglin_amd as B
    torch = torch_dev
    rng = np.random.default_rng(9)
    st = torch.cuda.Stream()
    c = B.Context(0, st.cuda_stream)
    S, nq, nk, D, page, wide = 3, 8, 2, 128, 16, 6
    dt = torch.bfloat16
    kv = [B.KVCache(S * wide, page, nk, D) for _ in range(2)]
    for x in kv:
        x.data.fill_(0xFF)
    table = torch.from_numpy(rng.permutation(S * wide).astype(np.int32).reshape(S, wide)).cuda()
    start = torch.arange(S + 1, dtype=torch.int32, device="cuda")
    qkv = torch.zeros((S, nq + 2 * nk, D), dtype=dt, device="cuda")
    q, k, v = qkv[:, :nq], qkv[:, nq:nq + nk], qkv[:, nq + nk:]
    lens, slots, pos = (torch.zeros(S, dtype=torch.int32, device="cuda") for _ in range(3))
    a = np.arange(512)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)
    rope = torch.from_numpy(np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)).cuda()
    outs = [(torch.empty((S, nq, D), dtype=dt, device="cuda"), torch.empty((S, nq, D), dtype=dt, device="cuda")) for _ in range(2)]

    def step(i):
        c.kv_append(kv[i], slots, k, v, q=q, q_out=outs[i][0], norm=B.NORM_RMS, rope=rope, pos=pos)
        c.attention(kv[i], outs[i][0], outs[i][1], start, lens, table, max_rows=1, max_len=wide * page)

    def inputs(n):
        ls = [n + 1 + 7 * s for s in range(S)]
        qkv.copy_(torch.from_numpy(rng.standard_normal(tuple(qkv.shape)).astype(np.float32)))
        lens.copy_(torch.tensor(ls, dtype=torch.int32))
        pos.copy_(torch.tensor([x - 1 for x in ls], dtype=torch.int32))
        slots.copy_(torch.tensor([int(table[s, (x - 1) // page]) * page + (x - 1) % page for s, x in enumerate(ls)], dtype=torch.int32))

    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        for n in range(-14, 0):                                                    # sequences 1 and 2 are longer: their first keys
            ls = [n + 1 + 7 * s for s in range(S)]
            if max(ls) < 1:
                continue
            inputs(n)
            slots.copy_(torch.where(lens > 0, slots, -1))
            lens.clamp_(min=0)
            pos.clamp_(min=0)
            step(0), step(1)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            step(0)
        for n in range(20):
            inputs(n)
            g.replay()
            step(1)
            st.synchronize()
            assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1]), n
            assert torch.isfinite(outs[0][1].float()).all()
    assert torch.equal(kv[0].data, kv[1].data)
    c.close()


def test_first_call_inside_a_capture_is_refused(torch_dev):
    import beglin_amd as B
    torch = torch_dev
    st = torch.cuda.Stream()
    c = B.Context(0, st.cuda_stream)
    kv = B.KVCache(2, 16, 1, 64)
    kv.data.zero_()
    q = torch.zeros((1, 1, 64), device="cuda")
    out = torch.zeros_like(q)
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    start, lens, table = i(0, 1), i(5), i(0, 1).reshape(1, 2)
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            with pytest.raises(B.BglError) as e:
                c.attention(kv, q, out, start, lens, table)
            assert e.value.code == B.E_CAPTURE
            q.zero_()
        st.synchronize()
    c.attention(kv, q, out, start, lens, table)
    c.close()
