"""Calls of bgl_attn_dev inside its limits that a count of all rows over the whole width of the table would refuse."""
import numpy as np
import pytest

import kv_forms as F
from test_gpu_attn import ctx, host, torch_dev  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs,window", [([(131072, 131072)], 50), ([(131072, 300)], 0), ([(131000, 300), (1, 400), (4, 90)], 0)], ids=str)
def test_long_prompts_over_wide_tables(torch_dev, ctx, seqs, window):  # noqa: F811
    """131072 rows of 64 heads over 8, a table for 2^20 keys."""
    import beglin_amd
    torch = torch_dev
    nq, nk, D, page, pages = 64, 8, 64, 4096, 3
    g = nq // nk
    gen = torch.Generator(device="cuda").manual_seed(1)
    cache = beglin_amd.KVCache(pages, page, nk, D)
    n = pages * page
    k, v = (torch.randn((n, nk, D), generator=gen, device="cuda") for _ in range(2))
    every = torch.arange(n, dtype=torch.int32, device="cuda")
    ctx.kv_append(cache, every, k, v)
    ctx.kv_read(cache, every, k, v)
    table = (torch.arange(1 << 20 >> 12, device="cuda") % pages).int()[None].repeat(len(seqs), 1)
    T = sum(r for r, _ in seqs)
    q = torch.randn((T, nq, D), generator=gen, device="cuda", dtype=torch.float16)
    out = torch.full_like(q, 7.0)
    start = np.concatenate([[0], np.cumsum([r for r, _ in seqs])]).astype(np.int32)
    lens = torch.tensor([m for _, m in seqs], dtype=torch.int32, device="cuda")
    ctx.attention(cache, q, out, torch.from_numpy(start).cuda(), lens, table, window=window, max_rows=max(r for r, _ in seqs))
    torch.cuda.synchronize()
    k, v, held = host(k), host(v), torch.from_numpy(start).tolist()
    for (r, m), at in zip(seqs, held):
        if r > m:
            assert int(out[at:at + r - m].count_nonzero()) == 0                    # rows before the first key
        first = max(0, r - min(m, 60))
        for i in sorted({first, max(first, r - 30)} | ({r // 2, 70} if window else set())):
            rows = np.arange(i, min(i + 30, r))
            lo = max(0, m - r + i - 60) if window else 0                           # the keys that these rows may see
            key = np.arange(lo, m if not window else m - r + rows[-1] + 1)
            pos = m - r + rows
            see = (key[None] <= pos[:, None]) & ((key[None] > pos[:, None] - window) if window else True)
            for h in (0, 13, nq - 1):
                F.attention_near(host(out[at + i:at + rows[-1] + 1, h]), host(q[at + i:at + rows[-1] + 1, h]), k[key % n, h // g], v[key % n, h // g], D ** -0.5, see,
                                 None, "float16", (at, i, h))


@pytest.mark.parametrize("rows", [1, 3, 50])
@pytest.mark.parametrize("window", [0, 20])
def test_lengths_outside_the_table(torch_dev, ctx, rows, window):  # noqa: F811
    """A length above ldt * page counts as ldt * page, one below 0 as 0."""
    import beglin_amd
    torch = torch_dev
    D, page, wide = 64, 16, 5
    cache = beglin_amd.KVCache(2 * wide, page, 2, D)
    n = 2 * wide * page
    ctx.kv_append(cache, torch.arange(n, dtype=torch.int32, device="cuda"), torch.randn((n, 2, D), device="cuda"), torch.randn((n, 2, D), device="cuda"))
    table = torch.arange(2 * wide, dtype=torch.int32, device="cuda").reshape(2, wide)
    q = torch.randn((2 * rows, 4, D), device="cuda")
    start = torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device="cuda")
    outs = []
    for lens in ((wide * page, 0), (wide * page + 7, -3), (2 ** 31 - 1, -2 ** 31)):
        out = torch.full_like(q, 7.0)
        ctx.attention(cache, q, out, start, torch.tensor(lens, dtype=torch.int32, device="cuda"), table, window=window, max_rows=rows)
        torch.cuda.synchronize()
        outs.append(out)
    assert torch.isfinite(outs[0]).all() and (outs[0][rows:] == 0).all() and (outs[0][:rows] != 0).any()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
