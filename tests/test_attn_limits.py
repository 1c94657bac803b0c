"""The limits of bgl_attn_dev (include/beglin_qgemv.h): calls past them are refused before any use of the context or the device."""
import ctypes as C

import pytest

import beglin_amd as B
from beglin_amd import capi
from test_attn_refusals import ATTN, KV, ctx, name, refused

WIDE = dict(ldt=1 << 20)                                    # pages of 32: 2^25 keys a sequence, 262149 units of a block of 16 rows
BAD = [dict(T=1 << 16, **WIDE),                             # 2 heads, 2^16 * 2 rows: 4.3e9 units
       dict(T=1 << 16, max_rows=16, **WIDE),
       dict(S=5000, T=6000, max_rows=1000, **WIDE),         # prompts and tokens: 5750 blocks, 3.0e9
       dict(T=1 << 27, max_rows=1 << 27)]                   # blocks of prompts


@pytest.mark.parametrize("change", BAD, ids=name)
def test_past_the_limits(change):
    kv, a = capi.bgl_kv(**KV), capi.bgl_attn(**{**ATTN, **change})
    refused(B.lib().bgl_attn_dev(ctx(), C.byref(kv), C.byref(a)), b"bgl_attn_dev")
