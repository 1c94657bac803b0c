"""fp32 rows of attention hold queries and weights in two fp16 parts each, 22 bits: within attn_bits' bound, which kernels with one part of either are
outside of at these sizes (test_attn_bits)."""
import numpy as np
import pytest

import attn_bits as A
from test_gpu_attn import ctx, host, torch_dev  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", A.CASES, ids=str)
def test_fp32_rows_hold_22_bits(torch_dev, ctx, case):  # noqa: F811
    import beglin_amd
    torch, (seqs, nq, nk, D) = torch_dev, case
    page, S = 16, len(seqs)
    wide = max(n for _, n in seqs) // page + 1
    cache = beglin_amd.KVCache(S * wide, page, nk, D)
    cache.data.fill_(0xFF)
    table = torch.arange(S * wide, dtype=torch.int32, device="cuda").reshape(S, wide)
    rows, k, v = [], [], []
    for s, (r, n) in enumerate(seqs):
        q, x, y = A.inputs(np.random.default_rng(100 * s + D), r, n, nq, nk, D)
        slots = torch.arange(n, dtype=torch.int32, device="cuda") + s * wide * page
        ctx.kv_append(cache, slots, torch.from_numpy(x).cuda(), torch.from_numpy(y).cuda())
        held = [torch.empty((n, nk, D), device="cuda") for _ in range(2)]
        ctx.kv_read(cache, slots, *held)
        torch.cuda.synchronize()
        rows.append(q), k.append(host(held[0])), v.append(host(held[1]))
    start = np.concatenate([[0], np.cumsum([r for r, _ in seqs])]).astype(np.int32)
    q = torch.from_numpy(np.concatenate(rows)).cuda()
    lens = torch.tensor([n for _, n in seqs], dtype=torch.int32, device="cuda")
    most, longest = max(r for r, _ in seqs), max(n for _, n in seqs)
    for hints in (dict(max_rows=most, max_len=longest), dict(max_rows=1, max_len=longest), dict(max_rows=most, max_len=10 ** 6)):
        out = torch.full_like(q, 7.0)
        ctx.attention(cache, q, out, torch.from_numpy(start).cuda(), lens, table, scale=A.SCALE, window=A.WINDOW, **hints)
        torch.cuda.synchronize()
        got = host(out)
        for s, (r, n) in enumerate(seqs):
            for h in range(nq):
                over = A.excess(got[start[s]:start[s] + r, h], rows[s][:, h], k[s][:, h * nk // nq], v[s][:, h * nk // nq], A.SCALE, A.seen(r, n))
                assert over <= 0, (hints, s, h, over)
