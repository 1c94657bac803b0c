"""Norms of heads without weights: w NULL is no factor, whatever w_add says (as bgl_norm_dev has it), for either of q and k by itself.

The fp32 arithmetic of 16-bit outputs and the double arithmetic of fp32 ones against the formula in 64 bits, within test_gpu_heads' bounds; the cache's
values are equal but for one code in 10^4 (a value on a border between codes)."""
import numpy as np
import pytest

import kv_forms as F
from test_gpu_heads import ctx, host, near, rope_table, rows, torch_dev  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 5, 700])
@pytest.mark.parametrize("norm", [1, 2])
@pytest.mark.parametrize("kind,out", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("style", [0, 1, 2])
def test_no_weights_are_no_factor(torch_dev, ctx, T, norm, kind, out, style):  # noqa: F811
    torch = torch_dev
    rng = np.random.default_rng(T + 10 * norm + style)
    D, nq, nk = 128, 30, 2
    q, k, v = rows(torch, rng, T, nq, D, kind), rows(torch, rng, T, nk, D, kind), rows(torch, rng, T, nk, D, kind)
    w = (0.2 * rng.standard_normal(D)).astype(np.float32)
    rope, pos = (rope_table(rng, 64, D), rng.integers(0, 64, T).astype(np.int32)) if style else (None, None)
    how = dict(norm=norm, eps=1e-5, w_add=1.0, rot=style, rope=torch.from_numpy(rope).cuda() if style else None,
               pos=torch.from_numpy(pos).cuda() if style else None)
    dt = getattr(torch, {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}[out])
    for qw, kw in ((None, None), (w, None), (None, w)):
        yq, yk = torch.empty(q.shape, dtype=dt, device="cuda"), torch.empty(k.shape, dtype=dt, device="cuda")
        both = [None if x is None else torch.from_numpy(x).cuda() for x in (qw, kw)]
        ctx.heads(q, k, yq, yk, q_w=both[0], k_w=both[1], **how)
        import beglin_amd
        cache = beglin_amd.KVCache(T // 16 + 1, 16, nk, D)
        slots, yc, gk = torch.arange(T, dtype=torch.int32, device="cuda"), torch.empty_like(yq), torch.empty(k.shape, dtype=torch.float16, device="cuda")
        ctx.kv_append(cache, slots, k, v, q=q, q_out=yc, q_w=both[0], k_w=both[1], **how)
        ctx.kv_read(cache, slots, gk)
        torch.cuda.synchronize()
        want = [F.heads(host(x), norm, y, 1e-5, 1.0, rope, pos, D, style) for x, y in ((q, qw), (k, kw))]
        near(yq, want[0], "q")
        near(yk, want[1], "k")
        near(yc, want[0], "q beside an append")
        assert (gk.cpu().numpy() != F.kept(want[1].astype(np.float32))).mean() <= 1e-4
