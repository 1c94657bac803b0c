"""Context.matmul_i8's own checks, on the CPU: what the library's entry cannot see behind a pointer is refused before the call.
The context has no handle, so a call that reaches the library is refused there, with another message."""
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


@pytest.mark.parametrize("ok", [dict(), dict(biases=None), dict(ys=torch.zeros((M, 64))[:, 3:3 + N]), dict(ys=torch.zeros((M, N), dtype=torch.bfloat16)),
                                dict(xq_dev=torch.zeros((M, 112), dtype=torch.int8)[:, :K])])
def test_allowed_calls_reach_the_library(ok):
    ctx, call = setting()
    with pytest.raises(B.BglError, match="bgl_matmul_i8_dev: bad argument"):
        ctx.matmul_i8(**{**call, **ok})
