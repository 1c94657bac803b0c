"""bgl_norm_dev's argument checks: they come before any use of the context or the device, so they run on the CPU (the
context here is a block of zeros that no check reads)."""
import ctypes as C

import pytest

import beglin_amd as B
from beglin_amd import capi

OK = dict(T=2, H=40, x=4096, ldx=40, x_type=B.T_F32, kind=B.NORM_RMS, eps=1e-6, y=1 << 20, ldy=40, y_type=B.T_F32, alpha=1.0)
BRANCH = dict(f=8192, ldf=40, f_type=B.T_F16, post=B.NORM_LAYER)
CODES = dict(yq=1 << 16, ldq=48, yscale=1 << 18)

BAD = [dict(T=0), dict(H=0), dict(T=-1), dict(x=None), dict(x_type=3), dict(x_type=-1), dict(y_type=9), dict(kind=3), dict(kind=-1),
       dict(post=B.NORM_RMS), dict(gate=4096), dict(y=None), dict(ldx=39), dict(ldy=39), dict(y=4096), dict(x_out=4096, ldo=48),
       dict(x_out=1 << 20, ldo=40), dict(x_out=1 << 21, ldo=39),
       dict(BRANCH, f_type=7), dict(BRANCH, post=4), dict(BRANCH, ldf=39), dict(BRANCH, x_out=8192, ldo=40), dict(BRANCH, y=8192),
       dict(BRANCH, gate=4096, gate_c=2), dict(BRANCH, gate=4096, gate_t=-1), dict(BRANCH, gate=4096, gate_t=39, gate_c=1),
       dict(BRANCH, gate=1 << 20, gate_c=1),
       dict(CODES, yscale=None), dict(yscale=4096), dict(CODES, ldq=40), dict(CODES, ldq=47), dict(CODES, ldq=32), dict(CODES, yq=(1 << 16) + 8)]


@pytest.mark.parametrize("change", BAD, ids=[" ".join(f"{k}={v}" for k, v in b.items()) for b in BAD])
def test_refused(change):
    ctx = C.create_string_buffer(1 << 14)
    d = capi.bgl_norm(**{**OK, **change})
    assert B.lib().bgl_norm_dev(ctx, C.byref(d)) == B.E_ARG
    assert b"bgl_norm_dev" in B.lib().bgl_last_error()


def test_null_arguments():
    d = capi.bgl_norm(**OK)
    assert B.lib().bgl_norm_dev(None, C.byref(d)) == B.E_ARG
    assert B.lib().bgl_norm_dev(C.create_string_buffer(1 << 14), None) == B.E_ARG
    assert B.lib().bgl_matmul_i8_dev(None, 1, None, None, 16, None, None, None, 0, None, 1) == B.E_ARG
