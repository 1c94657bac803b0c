"""A row's weights add up to 1: where every key has the same values, these are the output, whatever the scores.

A row's weights may be rounded to fp16 (2^-11 of each), but what divides their sum of values is their own sum.  So
out = v (1 + e), |e| <= (32 + n / 32 + 40) 2^-23 for the products' and sums' fp32 additions and the division: below 2^-16
for up to 2000 keys, where half a step of fp16 is 2^-12 of v at least: the fp16 output is the cached value itself, and a bf16 or fp32 one
within half a step, and e."""
import numpy as np
import pytest

import kv_forms as F
from test_gpu_attn import KINDS, ctx, host, torch_dev  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("keys", [2, 31, 700])
@pytest.mark.parametrize("rows", [1, 5, 40])
def test_equal_values_come_back(torch_dev, ctx, kind, D, keys, rows):  # noqa: F811
    import beglin_amd
    torch = torch_dev
    rng = np.random.default_rng(keys + D)
    S, nq, nk, page = 24, 4, 2, 16
    wide = (keys + rows + page - 1) // page
    cache = beglin_amd.KVCache(S * wide, page, nk, D)
    cache.data.fill_(0xFF)
    table = torch.arange(S * wide, dtype=torch.int32, device="cuda").reshape(S, wide)
    # key 0 scores highest, the others alike, so that their weights' roundings go the same way; a row's factor says by how much less
    n = keys + rows - 1
    k = np.zeros((S, n, nk, D), np.float32)
    k[..., 5] = 1.0
    k[:, 0, :, 5] = 2.0
    v = np.broadcast_to(1.99 + 0.009 * rng.random((S, 1, nk, D)), (S, n, nk, D)).astype(np.float32)
    at = np.arange(n)
    slots = torch.from_numpy((np.arange(S)[:, None] * wide * page + at).astype(np.int32).ravel()).cuda()
    ctx.kv_append(cache, slots, torch.from_numpy(k.reshape(-1, nk, D)).cuda(), torch.from_numpy(np.ascontiguousarray(v).reshape(-1, nk, D)).cuda())
    held = torch.empty((S * n, nk, D), dtype=torch.float16, device="cuda")
    ctx.kv_read(cache, slots, None, held)
    held = host(held).reshape(S, n, nk, D)
    assert (held == held[:, :1]).all()
    q = np.zeros((S, rows, nq, D), np.float32)
    q[..., 5] = rng.uniform(0.0, 6.0, (S, rows, nq))
    q = torch.from_numpy(q.reshape(-1, nq, D)).to(getattr(torch, KINDS[kind])).cuda()
    out = torch.full_like(q, 7.0)
    start = torch.arange(S + 1, dtype=torch.int32, device="cuda") * rows
    ctx.attention(cache, q, out, start, torch.full((S,), n, dtype=torch.int32, device="cuda"), table, scale=1.0, max_rows=rows, max_len=n)
    torch.cuda.synchronize()
    got = host(out).reshape(S, rows, nq, D)
    want = np.repeat(held[:, :1], nq // nk, 2).astype(np.float64)
    if kind == "f16":
        assert np.array_equal(got, np.broadcast_to(want, got.shape))
    e = (72 + n / 32) * 2.0 ** -23
    assert (np.abs(got - want) <= (F.HALF[KINDS[kind]] * (1 + e) + e) * np.abs(want)).all()
