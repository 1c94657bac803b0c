"""The bound of attn_bits tells operands of one fp16 part from two, for weights and for queries, at the sizes that test_gpu_attn_bits runs: a kernel
that dropped the second part of either would fail there."""
import numpy as np
import pytest

import attn_bits as A
import kv_forms as F


@pytest.mark.parametrize("case", A.CASES, ids=str)
def test_one_part_is_outside(case):
    seqs, nq, nk, D = case
    for s, (rows, keys) in enumerate(seqs):
        q, k, v = A.inputs(np.random.default_rng(100 * s + D), rows, keys, nq, nk, D)
        k, v, see = F.kept(k).astype(np.float32), F.kept(v).astype(np.float32), A.seen(rows, keys)
        worst = {}
        for parts in ((2, 2), (1, 2), (2, 1)):
            worst[parts] = [A.excess(A.emulate(q[:, h], k[:, h * nk // nq], v[:, h * nk // nq], A.SCALE, see, *parts), q[:, h], k[:, h * nk // nq],
                                     v[:, h * nk // nq], A.SCALE, see) for h in range(nq)]
        assert max(worst[2, 2]) <= 0
        if keys > 1:                                     # (one key: its weight is 1 whatever the score)
            assert max(worst[1, 2]) > 0 and max(worst[2, 1]) > 0
