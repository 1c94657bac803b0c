"""What Context.heads and Context.kv_append refuse before a call: tensors on the CPU, so that none gets through."""
import pytest
import torch

import beglin_amd as B


def context():
    c = B.Context.__new__(B.Context)
    c.h, c.device = None, -1                                       # the device of CPU tensors
    return c


def test_a_rotation_without_positions():
    c, x = context(), torch.zeros((3, 1, 64), dtype=torch.float16)
    kv = B.KVCache(2, 16, 1, 64, data=torch.zeros(2 * 20 * 64, dtype=torch.uint8))
    rope, slots = torch.zeros((5, 64)), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: c.heads(x, None, x.clone(), None, rope=rope), lambda: c.kv_append(kv, slots, x, x, rope=rope, rot=B.ROT_PAIRS)):
        with pytest.raises(B.BglError) as e:
            call()
        assert e.value.code == B.E_ARG
