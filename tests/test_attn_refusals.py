"""Argument checks of bgl_heads_dev, bgl_kv_append_dev, bgl_kv_read_dev and bgl_attn_dev: they come before any use of the context
or the device, so they run on the CPU (the context here is a block of zeros that no check reads)."""
import ctypes as C

import pytest

import beglin_amd as B
from beglin_amd import capi

ROPE = dict(rot_kind=B.ROT_HALF, rot=64, rope=1 << 22, n_pos=10, pos=1 << 23)
Q = dict(q=4096, ldq=512, hdq=128, q_out=1 << 20, ldqo=512, hdqo=128, nq=4)
K = dict(k=1 << 24, ldk=256, hdk=128, nk=2)
K_OUT = dict(k_out=1 << 25, ldko=256, hdko=128)
V = dict(v=1 << 26, ldv=256, hdv=128)
HEADS = dict(T=3, D=128, type=B.T_BF16, out_type=B.T_BF16, norm=B.NORM_RMS, eps=1e-6, **Q, **K, **K_OUT, **ROPE)
APPEND = {**{k: v for k, v in HEADS.items() if k not in K_OUT}, **V}
KV = dict(data=1 << 28, pages=8, page=32, heads=2, D=128)
ATTN = dict(S=2, T=3, nq=4, q=4096, ldq=512, hdq=128, out=1 << 20, ldo=512, hdo=128, type=B.T_F16, start=1 << 21, len=1 << 22,
            table=1 << 23, ldt=4, scale=0.1, causal=1, max_rows=1, max_len=100)

BAD_HEADS = [dict(T=0), dict(T=-1), dict(D=0), dict(D=12), dict(D=520), dict(type=3), dict(type=-1), dict(out_type=3), dict(norm=3), dict(norm=-1),
             dict(rot_kind=3), dict(rot_kind=-1), dict(rope=None), dict(pos=None), dict(n_pos=0), dict(rot=0), dict(rot=8), dict(rot=72),
             dict(rot=144), dict(rot_kind=B.ROT_PAIRS, rot=4), dict(rot_kind=B.ROT_PAIRS, rot=20), dict(q=None), dict(q_out=None),
             dict(k=None), dict(k_out=None), dict(nq=0), dict(nq=70000), dict(nk=0), dict(ldq=511), dict(hdq=127), dict(ldq=-512), dict(ldqo=500),
             dict(ldk=200), dict(hdk=100), dict(ldko=1), dict(hdko=-128), dict(v=1 << 26), dict(q=None, k=None, q_out=None, k_out=None),
             dict(q_out=4096, ldqo=600), dict(q_out=4096, out_type=B.T_F32), dict(k_out=1 << 24, hdko=256, ldko=640), dict(q_out=1 << 24),
             dict(k_out=4096), dict(k_out=1 << 20)]
BAD_APPEND = [dict(T=0), dict(k=None), dict(v=None), dict(k_out=1 << 25, ldko=256, hdko=128), dict(nk=3, ldk=384, ldv=384), dict(D=64, rot=64),
              dict(ldv=100), dict(hdv=64), dict(q_out=None), dict(q_out=1 << 26), dict(type=4), dict(rot=100)]
BAD_KV = [dict(data=None), dict(data=(1 << 28) + 8), dict(pages=0), dict(page=0), dict(page=24), dict(page=8), dict(page=-16), dict(heads=0),
          dict(D=80), dict(D=0), dict(D=512), dict(pages=1 << 27, page=32)]
BAD_ATTN = [dict(S=0), dict(T=0), dict(ldt=0), dict(nq=0), dict(nq=3), dict(nq=-2), dict(q=None), dict(out=None), dict(start=None), dict(len=None),
            dict(table=None), dict(type=5), dict(ldq=300), dict(hdq=64), dict(ldo=300), dict(hdo=-1), dict(window=-1),
            dict(window=5, causal=0), dict(max_rows=-1), dict(max_len=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(out=4096),
            dict(T=1 << 30, nq=8, ldq=1024, ldo=1024), dict(ldt=(1 << 25) + 1), dict(ldt=1 << 30),
            dict(T=1 << 25, nq=32, ldq=4096, ldo=4096, max_rows=1 << 25)]


def name(b):
    return " ".join(f"{k}={v}" for k, v in b.items())


def ctx():
    return C.create_string_buffer(1 << 14)


def refused(rc, who):
    assert rc == B.E_ARG
    assert who in B.lib().bgl_last_error()


@pytest.mark.parametrize("change", BAD_HEADS, ids=name)
def test_heads_refused(change):
    d = capi.bgl_heads(**{**HEADS, **change})
    refused(B.lib().bgl_heads_dev(ctx(), C.byref(d)), b"bgl_heads_dev")


@pytest.mark.parametrize("change", BAD_APPEND, ids=name)
def test_append_refused(change):
    kv, d = capi.bgl_kv(**KV), capi.bgl_heads(**{**APPEND, **change})
    refused(B.lib().bgl_kv_append_dev(ctx(), C.byref(kv), C.byref(d), 1 << 27), b"bgl_kv_append_dev")


@pytest.mark.parametrize("change", BAD_KV, ids=name)
def test_cache_refused(change):
    kv, d, a = capi.bgl_kv(**{**KV, **change}), capi.bgl_heads(**APPEND), capi.bgl_attn(**ATTN)
    refused(B.lib().bgl_kv_append_dev(ctx(), C.byref(kv), C.byref(d), 1 << 27), b"bgl_kv_append_dev")
    refused(B.lib().bgl_kv_read_dev(ctx(), C.byref(kv), 1 << 27, 3, 4096, 256, 128, None, 0, 0, B.T_F32), b"bgl_kv_read_dev")
    refused(B.lib().bgl_attn_dev(ctx(), C.byref(kv), C.byref(a)), b"bgl_attn_dev")


@pytest.mark.parametrize("change", BAD_ATTN, ids=name)
def test_attn_refused(change):
    kv, a = capi.bgl_kv(**KV), capi.bgl_attn(**{**ATTN, **change})
    refused(B.lib().bgl_attn_dev(ctx(), C.byref(kv), C.byref(a)), b"bgl_attn_dev")


def test_read_refused():
    kv = capi.bgl_kv(**KV)
    read = lambda slots=1 << 27, n=3, k=4096, ldk=256, hdk=128, v=1 << 20, ldv=256, hdv=128, t=B.T_F16: B.lib().bgl_kv_read_dev(  # noqa: E731
        ctx(), C.byref(kv), slots, n, k, ldk, hdk, v, ldv, hdv, t)
    for bad in (dict(slots=None), dict(n=0), dict(k=None, v=None), dict(ldk=100), dict(hdv=64), dict(t=3), dict(v=4096)):
        refused(read(**bad), b"bgl_kv_read_dev")


def test_null_arguments():
    kv, d, a = capi.bgl_kv(**KV), capi.bgl_heads(**HEADS), capi.bgl_attn(**ATTN)
    L = B.lib()
    assert L.bgl_heads_dev(None, C.byref(d)) == B.E_ARG and L.bgl_heads_dev(ctx(), None) == B.E_ARG
    for bad in ((None, C.byref(kv), C.byref(d), 64), (ctx(), None, C.byref(d), 64), (ctx(), C.byref(kv), None, 64), (ctx(), C.byref(kv), C.byref(d), None)):
        assert L.bgl_kv_append_dev(*bad) == B.E_ARG
    for bad in ((None, C.byref(kv), C.byref(a)), (ctx(), None, C.byref(a)), (ctx(), C.byref(kv), None)):
        assert L.bgl_attn_dev(*bad) == B.E_ARG


def test_cache_bytes():
    L = B.lib()
    assert L.bgl_kv_bytes(7, 48, 5, 96) == 7 * 5 * 3 * 20 * 96
    assert L.bgl_kv_bytes(1 << 20, 64, 8, 128) == (1 << 20) * 8 * 4 * 20 * 128          # past 32 bits
    for bad in ((0, 16, 1, 64), (1, 8, 1, 64), (1, 20, 1, 64), (1, 16, 0, 64), (1, 16, 1, 32), (1 << 28, 16, 1, 64)):
        assert L.bgl_kv_bytes(*bad) == 0


def test_python_checks():
    """What the entries cannot see behind a pointer; tensors on the CPU, so that no call gets through."""
    import torch

    def context():
        c = B.Context.__new__(B.Context)
        c.h, c.device = None, -1                                   # the device of CPU tensors
        return c
    c = context()
    with pytest.raises(B.BglError):
        B.KVCache(2, 24, 1, 64)
    with pytest.raises(B.BglError):
        B.KVCache(2, 16, 1, 64, data=torch.zeros(5, dtype=torch.uint8))
    kv = B.KVCache(2, 16, 1, 64, data=torch.zeros(2 * 20 * 64, dtype=torch.uint8))
    f = lambda *s, t=torch.float16: torch.zeros(s, dtype=t)  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    x = f(3, 1, 64)
    ok = dict(start=i(3), lens=i(2), table=i(2, 4))
    bad = [dict(q=f(3, 64), out=x, **ok), dict(q=f(3, 1, 96), out=f(3, 1, 96), **ok), dict(q=x, out=f(2, 1, 64), **ok), dict(q=x, out=x.float(), **ok),
           dict(q=x, out=x.clone(), start=i(2), lens=i(2), table=i(2, 4)), dict(q=x, out=x.clone(), start=i(3), lens=i(3), table=i(2, 4)),
           dict(q=x, out=x.clone(), start=i(3).long(), lens=i(2), table=i(2, 4)), dict(q=x, out=x.clone(), start=i(3), lens=i(2), table=i(8)),
           dict(q=x, out=x.clone(), start=i(3), lens=i(2), table=i(4, 2).t()), dict(q=x.double(), out=x.double(), **ok),
           dict(q=x, out=x.clone(), sink=f(1), **ok), dict(q=x, out=x.clone(), sink=f(2, t=torch.float32), **ok),
           dict(q=f(3, 64, 1).transpose(1, 2), out=x, **ok)]
    bad[-1]["q"] = torch.zeros((3, 1, 128), dtype=torch.float16)[:, :, ::2]
    for b in bad:
        with pytest.raises(B.BglError) as e:
            c.attention(kv, **b)
        assert e.value.code == B.E_ARG
    s = i(3)
    for args, more in (((s, x, x.float()), {}), ((s, x, f(2, 1, 64)), {}), ((i(2), x, x), {}), ((s.long(), x, x), {}), ((s, x, x), dict(q=x)),
                       ((s, f(3, 2, 64), f(3, 1, 64)), {}), ((s, x, x), dict(rope=f(5, 64), pos=i(3))),
                       ((s, x, x), dict(rope=f(5, 64, t=torch.float32), pos=i(2))), ((s, x, x), dict(norm=1, k_w=f(63, t=torch.float32)))):
        with pytest.raises(B.BglError):
            c.kv_append(kv, *args, **more)
    for args in ((None, None, None, None), (x, None, None, None), (None, x, None, None), (x, x, x, x.float()), (x, f(2, 1, 64), x, f(2, 1, 64)), (f(3, 64), None, x, None)):
        with pytest.raises(B.BglError):
            c.heads(*args)
    for args in ((s, None, None), (s, f(2, 1, 64), None), (s, x, x.float()), (s.long(), x, None)):
        with pytest.raises(B.BglError):
            c.kv_read(kv, *args)
