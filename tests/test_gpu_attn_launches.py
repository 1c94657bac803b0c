"""Sequences of few rows beside prompts: one launch or two, by what each costs as far as the call's hints tell (us measured, 32 heads over 8)."""
import pytest

from test_gpu_attn import Batch, ctx, torch_dev  # noqa: F401

pytestmark = pytest.mark.gpu
CASES = [  # rows of each sequence, D, type, max_len, window, launches             us in one launch, in two
    ([200] + [1] * 15, 128, "bf16", 1000, 0, 1),                                   # 29, 45
    ([100] + [1] * 3, 64, "f16", 2000, 0, 1),                                      # 19, 31 (a prompt of 100 keys: 15, 25)
    ([500] + [1] * 20, 128, "bf16", 500, 0, 1),                                    # 20, 28 (300 keys)
    ([40] + [1] * 31, 128, "bf16", 4000, 512, 1),                                  # 20, 34
    ([40] + [1] * 31, 256, "bf16", 2048, 0, 2),                                    # 179, 85 (a prompt of 40 keys: 102, 59)
    ([40] + [1] * 31, 128, "f32", 2048, 0, 2),                                     # 154, 78 (85, 57)
    ([40] + [1] * 15, 256, "bf16", 2000, 0, 2),                                    # (91, 48)
    ([2000] + [1] * 31, 128, "bf16", 3000, 0, 2),                                  # 147, 130
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_launches(torch_dev, ctx, case):  # noqa: F811
    rows, D, kind, longest, window, launches = case
    b = Batch(torch_dev, ctx, [(r, r + 3) for r in rows], 32, 8, D, kind, 64)
    ctx.prof_enable(True)
    ctx.prof_read()
    got = b.run(ctx, max_rows=max(rows), max_len=longest, window=window)
    assert sum(v[1] for v in ctx.prof_read().values()) == launches
    ctx.prof_enable(False)
    b.check(got, window=window, only=[s for s in range(len(rows)) if rows[s] < 300])
