"""Pages whose part of one head is longer than 2^32 bytes: keys at their end, for single rows and prompts."""
import numpy as np
import pytest

import kv_forms as F
from test_gpu_attn import ctx, host, torch_dev  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 40, 300])
@pytest.mark.parametrize("kind", ["bfloat16", "float32"])
def test_keys_past_4_gib_in_a_page(torch_dev, ctx, rows, kind):  # noqa: F811
    import beglin_amd
    torch = torch_dev
    D, nq, window, n = 256, 2, 100, 500
    page = 838900 * 16                                                             # records of 5120 bytes: 39 of them past 2^32
    cache = beglin_amd.KVCache(1, page, 1, D)
    cache.data.zero_()
    rng = np.random.default_rng(rows)
    k, v = (torch.from_numpy(rng.standard_normal((n, 1, D)).astype(np.float32)).cuda() for _ in range(2))
    slots = torch.arange(page - n, page, dtype=torch.int32, device="cuda")
    ctx.kv_append(cache, slots, k, v)
    ctx.kv_read(cache, slots, k, v)
    q = torch.from_numpy(rng.standard_normal((rows, nq, D)).astype(np.float32)).cuda().to(getattr(torch, kind))
    out = torch.full_like(q, 7.0)
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    ctx.attention(cache, q, out, i(0, rows), i(page), i(0)[None], window=window, max_rows=rows, max_len=page)
    torch.cuda.synchronize()
    pos, key = np.arange(n - rows, n)[:, None], np.arange(n)[None]
    see = (key <= pos) & (key > pos - window)
    for h in range(nq):
        F.attention_near(host(out[:, h]), host(q[:, h]), host(k[:, 0]), host(v[:, 0]), D ** -0.5, see, None, kind, h)
    del cache
    torch.cuda.empty_cache()
