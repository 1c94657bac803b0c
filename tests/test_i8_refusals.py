"""The checks of Context.matmul_i8, Context.norm and Context.bind, on the CPU: what the library's entries cannot see behind a pointer is
refused before the call.  The context has no handle, so a call that reaches the library is refused there, with another
message."""
import pytest
import torch

import beglin_amd as B

M, N, K = 3, 40, 100


def setting():
    ctx = B.Context.__new__(B.Context)
    ctx.h, ctx.device = None, -1                            # -1: where the tensors of this file lie
    t = B.Tensor(1)
    t._shape = (N, K)
    return ctx, dict(ts=t, xq_dev=torch.zeros((M, 112), dtype=torch.int8), ascale_dev=torch.zeros(M), ys=torch.zeros((M, N)), biases=torch.zeros(N))


BAD = {
    "a view of fewer channels": dict(ys=torch.zeros((M, 64))[:, :N - 1]),
    "a view of more channels": dict(ys=torch.zeros((M, 64))),
    "fewer rows of y": dict(ys=torch.zeros((M - 1, N))),
    "more rows of y": dict(ys=torch.zeros((M + 1, N))),
    "y of one dimension": dict(ys=torch.zeros(M * N)),
    "rows of y that are not dense": dict(ys=torch.zeros((M, 2 * N))[:, ::2]),
    "y of another type": dict(ys=torch.zeros((M, N), dtype=torch.float64)),
    "a short bias": dict(biases=torch.zeros(N - 1)),
    "a bias of 16 bits": dict(biases=torch.zeros(N, dtype=torch.float16)),
    "a bias with gaps": dict(biases=torch.zeros(2 * N)[::2]),
    "few scales": dict(ascale_dev=torch.zeros(M - 1)),
    "scales of 16 bits": dict(ascale_dev=torch.zeros(M, dtype=torch.bfloat16)),
    "scales with gaps": dict(ascale_dev=torch.zeros(2 * M)[::2]),
    "codes of one dimension": dict(xq_dev=torch.zeros(112, dtype=torch.int8)),
    "codes of another type": dict(xq_dev=torch.zeros((M, 112), dtype=torch.uint8)),
    "codes of fewer inputs": dict(xq_dev=torch.zeros((M, 128), dtype=torch.int8)[:, :K - 1]),
    "a last row that ends with the allocation": dict(xq_dev=torch.zeros(M * 112 - 12, dtype=torch.int8).as_strided((M, K), (112, 1))),
}


@pytest.mark.parametrize("change", BAD.values(), ids=list(BAD))
def test_refused(change):
    ctx, call = setting()
    with pytest.raises(B.BglError, match="matmul_i8:") as e:
        ctx.matmul_i8(**{**call, **change})
    assert e.value.code == B.E_ARG


def test_tensors_of_another_device():
    ctx, call = setting()
    ctx.device = 0
    with pytest.raises(B.BglError, match="device 0"):
        ctx.matmul_i8(**call)


def test_groups():
    ctx, call = setting()
    call["ts"], call["ys"], call["biases"] = [call["ts"]] * 2, [call["ys"], torch.zeros((M, N), dtype=torch.float16)], None
    with pytest.raises(B.BglError, match="matmul_i8: y is"):
        ctx.matmul_i8(**call)                               # two types
    call["ys"] = call["ys"][:1]
    with pytest.raises(B.BglError, match="matmul_i8: one y"):
        ctx.matmul_i8(**call)
    call["ts"], call["ys"] = [], []
    with pytest.raises(B.BglError, match="matmul_i8: one y"):
        ctx.matmul_i8(**call)


@pytest.mark.parametrize("ok", [dict(), dict(biases=None), dict(ascale_dev=torch.zeros((M, 1)), biases=torch.zeros((1, N))), dict(ys=torch.zeros((M, 64))[:, 3:3 + N]), dict(ys=torch.zeros((M, N), dtype=torch.bfloat16)),
                                dict(xq_dev=torch.zeros((M, 112), dtype=torch.int8)[:, :K])])
def test_allowed_calls_reach_the_library(ok):
    ctx, call = setting()
    with pytest.raises(B.BglError, match="bgl_matmul_i8_dev: bad argument"):
        ctx.matmul_i8(**{**call, **ok})


T, H = 3, 40


def norm_call(**change):
    ctx, _ = setting()
    ctx.device = change.pop("device", -1)
    x = change.pop("x", torch.zeros((T, H)))
    ctx.norm(x, **{**dict(yq=torch.zeros((T, 48), dtype=torch.int8), yscale=torch.zeros(T)), **change})


NORM_BAD = {
    "a view that ends inside 16 codes": dict(yq=torch.zeros((T, 64), dtype=torch.int8)[:, :47]),
    "a view of the last columns": dict(yq=torch.zeros((T, 64), dtype=torch.int8)[:, 48:]),
    "rows of H codes": dict(yq=torch.zeros((T, H), dtype=torch.int8)),
    "fewer rows": dict(yq=torch.zeros((T - 1, 48), dtype=torch.int8)),
    "codes of another type": dict(yq=torch.zeros((T, 48), dtype=torch.uint8)),
    "rows that are not dense": dict(yq=torch.zeros((T, 96), dtype=torch.int8)[:, ::2]),
    "one dimension": dict(yq=torch.zeros(T * 48, dtype=torch.int8)),
    "few scales": dict(yscale=torch.zeros(T - 1)), "no scales": dict(yscale=None), "another device": dict(device=0),
}


@pytest.mark.parametrize("change", NORM_BAD.values(), ids=list(NORM_BAD))
def test_norm_refused(change):
    with pytest.raises(B.BglError, match="norm: ") as e:
        norm_call(**dict(change))
    assert e.value.code == B.E_ARG


def test_norm_calls_reach_the_library():
    for ok in (dict(), dict(w=torch.zeros(H), b=torch.zeros((1, H)), branch=torch.zeros((T, 64))[:, :H], branch_kind=B.NORM_RMS, branch_w=torch.zeros(H),
                            gate=torch.zeros((1, H)), x_out=torch.zeros((T, H))), dict(yq=torch.zeros((T, 96), dtype=torch.int8)[:, 16:64]), dict(yq=None, yscale=None, y=torch.zeros((T, H)))):
        with pytest.raises(B.BglError, match="bgl_norm_dev: NULL"):
            norm_call(**ok)


@pytest.mark.parametrize("codes,scales", [
    (torch.zeros((4, 8), dtype=torch.int8), torch.zeros(3)), (torch.zeros((4, 8), dtype=torch.int8), torch.zeros(4, dtype=torch.float16)),
    (torch.zeros((4, 7), dtype=torch.int8), torch.zeros(4)), (torch.zeros((4, 8)), torch.zeros(4)),
    (torch.zeros((4, 16), dtype=torch.int8)[:, ::2], torch.zeros(4))],
    ids=["few scales", "scales of 16 bits", "few codes", "codes of another type", "codes with gaps"])
def test_bind_refused(codes, scales):
    ctx, _ = setting()
    with pytest.raises(B.BglError, match="bind:") as e:
        ctx.bind(B.K_Q8C, codes, scales, 4, 8)
    assert e.value.code == B.E_ARG


def test_bind_of_torch_tensors_reaches_the_library():
    ctx, _ = setting()
    for codes, scales in ((torch.zeros((4, 8), dtype=torch.int8), torch.zeros(4)), (torch.zeros((4, 8), dtype=torch.int8).numpy(), torch.zeros(4).numpy())):
        with pytest.raises(B.BglError, match="bgl_bind: NULL"):
            ctx.bind(B.K_Q8C, codes, scales, 4, 8)
