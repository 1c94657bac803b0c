"""beglin_amd -- MI355X (gfx950) backend for beglin's quantized GEMV / MoE-gather hot path.

The product is the C-ABI library libbeglin_hip.so (include/beglin_qgemv.h).  This package is a
thin Python veneer over it for tests and benchmarks: PyTorch only supplies device memory and the
stream.  Every call goes through the HIP library; if it is not built, importing `Context` fails.
"""
import ctypes as C

from . import capi
from .capi import (ACT_F32, ACT_W4A8, K_F16, K_F32, K_MXFP4, K_Q4G32H, K_Q4G64, K_Q4G64A,  # noqa: F401
                   K_Q4G256P, K_Q4G256SF, K_Q8C, K_Q8G64, K_QNG64, NORM_LAYER, NORM_NONE, NORM_RMS,
                   ROT_HALF, ROT_NONE, ROT_PAIRS, T_BF16, T_F16, T_F32)

_lib = None


def lib():
    global _lib
    if _lib is None:
        _lib = capi.load()
    return _lib


# BGL_E_* codes of include/beglin_qgemv.h
E_ARG, E_UNSUPPORTED, E_HIP, E_NODEV, E_NOMEM, E_CAPTURE, E_TIMEOUT = -1, -2, -3, -4, -5, -6, -7


class BglError(RuntimeError):
    def __init__(self, msg, code=0):
        super().__init__(msg)
        self.code = code


def _check(rc, what):
    if rc != 0:
        raise BglError(f"{what} failed ({rc}): {lib().bgl_last_error().decode(errors='replace')}", rc)


def _p(t):
    """Device (or host numpy) pointer of a torch tensor / numpy array, None passes through."""
    if t is None:
        return None
    if hasattr(t, "data_ptr"):
        assert t.is_contiguous(), "tensor must be contiguous"
        return C.c_void_p(t.data_ptr())
    return C.c_void_p(t.ctypes.data)


_DT = None


def _dtypes():
    """torch's fp32, fp16, bf16 (at their BGL_T_* places) and int8."""
    global _DT
    if _DT is None:
        import torch
        _DT = (torch.float32, torch.float16, torch.bfloat16, torch.int8)
    return _DT


def _type(t):
    return _dtypes().index(t.dtype, 0, 3)


def _rows(t, T, H, dev):
    """Pointer and distance in elements of the dense rows of a [T][H] tensor on device dev."""
    assert t.shape == (T, H), "rows must be [T][H]"
    ld, one = t.stride()
    assert one == 1 or H == 1, "rows must be dense"
    if t.get_device() != dev:
        _refuse(f"norm: tensors lie on device {dev}")
    return t.data_ptr(), ld if T > 1 else H


def _vec(t, n, dev):
    """Pointer of an fp32 vector of n values on device dev, None passes through."""
    if t is None:
        return None
    assert t.dtype is _dtypes()[0] and t.numel() == n and t.is_contiguous(), "fp32 vector expected"
    if t.get_device() != dev:
        _refuse(f"norm: tensors lie on device {dev}")
    return t.data_ptr()


def _w(t):
    """Address of a weight buffer to bind: a numpy array, or a torch tensor in host or device memory; None passes through."""
    return None if t is None else t.data_ptr() if hasattr(t, "data_ptr") else t.ctypes.data


def _refuse(what):
    """Refuses a call as the library does, for what its entries cannot see behind a pointer.  (The checks of the calls of a
    step are written to take no more than the rest of a call: a small product takes 8 us, and so does its host side.)"""
    raise BglError(what, E_ARG)


_ARRAYS = {}


def _arrays(n):
    """Arrays for n tensors, outputs, biases (all NULL) and row strides."""
    if n not in _ARRAYS:
        _ARRAYS[n] = C.c_void_p * n, C.c_long * n
    p, l = _ARRAYS[n]
    return p(), p(), p(), l()


def _weights(kind, out, inn, packed, scales, sub):
    """What a bind reads of torch tensors: dense ones, scales of the kind's type, and K_Q8C's buffers whole."""
    for t in (packed, scales, sub):
        if hasattr(t, "data_ptr") and not t.is_contiguous():
            _refuse("bind: torch tensors have to be dense")
    if hasattr(scales, "data_ptr"):
        if not (scales.element_size() == 2 if kind == K_Q4G32H else scales.dtype is _dtypes()[0]):
            _refuse("bind: scales of another type")
        if kind == K_Q8C and scales.numel() != out:
            _refuse(f"bind: K_Q8C takes scales [out={out}]")
    if kind == K_Q8C and hasattr(packed, "data_ptr") and not (packed.dtype is _dtypes()[3] and packed.numel() == out * inn):
        _refuse(f"bind: K_Q8C takes int8 codes [{out}][{inn}]")


class Tensor:
    """A weight tensor bound on the device (bgl_tensor*)."""

    def __init__(self, handle):
        self.h = C.c_void_p(handle) if not isinstance(handle, C.c_void_p) else handle
        self._shape = None

    def shape(self):
        """(out, in), asked of the library once."""
        if self._shape is None:
            i = self.info()
            self._shape = i["out"], i["inn"]
        return self._shape

    def info(self):
        k, b, o, i = C.c_int(), C.c_int(), C.c_int(), C.c_int()
        nb = C.c_size_t()
        _check(lib().bgl_tensor_info(self.h, C.byref(k), C.byref(b), C.byref(o), C.byref(i), C.byref(nb)), "bgl_tensor_info")
        return dict(kind=k.value, bits=b.value, out=o.value, inn=i.value, device_bytes=nb.value)

    def free(self):
        if self.h:
            lib().bgl_tensor_free(self.h)
            self.h = None


def _heads(t, shape, kind, dev, who):
    """Pointer and distances in elements between the tokens and the heads of a [T][heads][D] tensor of a type on device dev."""
    if t.shape != shape or t.dtype is not kind or t.get_device() != dev:
        _refuse(f"{who}: heads are {kind} {tuple(shape)} on device {dev}")
    ld, hd, one = t.stride()
    if one != 1:
        _refuse(f"{who}: the values of a head are dense")
    return t.data_ptr(), ld, hd


def _row_type(kind, who):
    d = _dtypes()
    return T_F32 if kind is d[0] else T_F16 if kind is d[1] else T_BF16 if kind is d[2] else _refuse(f"{who}: rows are fp32, fp16 or bf16")


_INT32 = None
_NO_ROWS = None, 0, 0


def _ints(t, n, dev, who):
    """Pointer of a dense int32 vector of n values on device dev."""
    global _INT32
    if _INT32 is None:
        import torch
        _INT32 = torch.int32
    if t.dtype is not _INT32 or t.numel() != n or t.get_device() != dev or not t.is_contiguous():
        _refuse(f"{who}: int32 [{n}] on device {dev} expected")
    return t.data_ptr()


def _floats(t, n, dev, who):
    """Pointer of a dense fp32 vector of n values on device dev, None passes through."""
    if t is None:
        return None
    if t.dtype is not _dtypes()[0] or t.numel() != n or t.get_device() != dev or not t.is_contiguous():
        _refuse(f"{who}: fp32 [{n}] on device {dev} expected")
    return t.data_ptr()


class KVCache:
    """A paged cache of keys and values in 4 bits (bgl_kv): `pages` pages of `page` tokens (a multiple of 16), `heads` heads of `dim`
    values.  data: the uint8 buffer to use (dense, bgl_kv_bytes long); made on the device if None."""

    def __init__(self, pages, page, heads, dim, data=None, device=0):
        import torch
        n = lib().bgl_kv_bytes(pages, page, heads, dim)
        if not n:
            _refuse(f"KVCache: no cache of {pages} pages of {page} tokens (a multiple of 16), {heads} heads of {dim} values "
                    "(64, 96, 128, 192, 256)")
        if data is None:
            data = torch.empty(n, dtype=torch.uint8, device=f"cuda:{device}")
        if data.dtype is not torch.uint8 or data.numel() != n or not data.is_contiguous():
            _refuse(f"KVCache: data is a dense uint8 buffer of {n} bytes")
        self.data, self.pages, self.page, self.heads, self.dim = data, pages, page, heads, dim
        self.device = data.get_device()
        self.d = capi.bgl_kv(data.data_ptr(), pages, page, heads, dim)


class Context:
    """One bgl_ctx on one device and one HIP stream (torch's current stream by default)."""

    def __init__(self, device=0, stream=None):
        import torch
        L = lib()
        if stream is None:
            stream = torch.cuda.current_stream(device).cuda_stream
        h = C.c_void_p()
        _check(L.bgl_ctx_create(device, C.c_void_p(stream), C.byref(h)), "bgl_ctx_create")
        self.h = h
        self.device = device

    def close(self):
        if self.h:
            lib().bgl_ctx_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def sync(self):
        _check(lib().bgl_synchronize(self.h), "bgl_synchronize")

    def check(self):
        """Synchronize, then raise if a bounded in-kernel wait gave up since the last check (bgl_ctx_check)."""
        _check(lib().bgl_ctx_check(self.h), "bgl_ctx_check")

    # ---- profiling (QWEN_PROF analogue) ----
    def prof_enable(self, on=True):
        _check(lib().bgl_prof_enable(self.h, int(on)), "bgl_prof_enable")

    def prof_read(self):
        """{phase: (ms, launches)} for phases prep/gemv/other, summed since the last read."""
        ms = (C.c_double * 3)()
        n = (C.c_int * 3)()
        _check(lib().bgl_prof_read(self.h, ms, n, 3), "bgl_prof_read")
        return {"prep": (ms[0], n[0]), "gemv": (ms[1], n[1]), "other": (ms[2], n[2])}

    # ---- binding ----
    def bind(self, kind, packed, scales, out, inn, bits=0, sub=None):
        """Bind buffers in the reference layout (sub: g256sf sub-codes or Q4G64A biases; scales None for the dense
        kinds and MXFP4, whose blocks carry their exponents): numpy arrays, or dense torch tensors in host memory or on
        the device, where the context's stream has to see them written."""
        _weights(kind, out, inn, packed, scales, sub)
        w = capi.bgl_wt(kind, bits if kind == K_QNG64 else (8 if kind in (K_Q8G64, K_Q8C) else 4), out, inn,
                        _w(packed), _w(scales), _w(sub))
        h = C.c_void_p()
        _check(lib().bgl_bind(self.h, C.byref(w), C.byref(h)), "bgl_bind")
        return Tensor(h)

    def bind_qng64_mixed(self, planes, offsets, bits, scales, out, inn):
        """Bind a mixed per-cell qNg64 tensor (numpy planes u8, offsets u32 [cells+1], bits u8 [cells],
        scales f32 [cells])."""
        h = C.c_void_p()
        _check(lib().bgl_bind_qng64_mixed(self.h, planes.ctypes.data, planes.nbytes, offsets.ctypes.data, bits.ctypes.data,
                                          scales.ctypes.data, out, inn, C.byref(h)), "bgl_bind_qng64_mixed")
        return Tensor(h)

    def quantize(self, kind, w_dev, bits=0, qng64_encoder=1, want_ref=False):
        """Quantize fp32 weights already on the device (torch tensor [out][in]).  With want_ref the
        reference-layout bytes come back as numpy arrays."""
        import numpy as np
        out, inn = w_dev.shape
        ref = None
        args = [None, None, None]
        if want_ref:
            if kind in (K_Q4G64, K_Q4G256SF, K_Q4G32H):
                pk = np.zeros((out, inn // 2), np.uint8)
            elif kind in (K_Q8G64, K_Q8C):
                pk = np.zeros((out, inn), np.int8)
            else:
                pk = np.zeros((out, inn // 64 * bits * 8), np.uint8)
            if kind == K_Q4G32H:
                sc = np.zeros((out, inn // 32), np.uint16)
            elif kind == K_Q4G256SF:
                sc = np.zeros((out, inn // 256), np.float32)
            elif kind == K_Q8C:
                sc = np.zeros(out, np.float32)
            else:
                sc = np.zeros((out, inn // 64), np.float32)
            sub = np.zeros((out, inn // 64), np.uint8) if kind == K_Q4G256SF else None
            ref = (pk, sc, sub)
            args = [_p(pk), _p(sc), _p(sub)]
        h = C.c_void_p()
        _check(lib().bgl_quantize_dev(self.h, kind, bits, int(qng64_encoder), _p(w_dev), out, inn, C.byref(h), *args),
               "bgl_quantize_dev")
        return (Tensor(h), ref) if want_ref else Tensor(h)

    def dequant(self, t, row0, nrows, out_dev):
        _check(lib().bgl_dequant_dev(self.h, t.h, row0, nrows, _p(out_dev)), "bgl_dequant_dev")

    # ---- compute (device pointers) ----
    def matmul(self, t, x_dev, y_dev, act=ACT_F32, bias_dev=None):
        M = 1 if x_dev.dim() == 1 else x_dev.shape[0]
        _check(lib().bgl_matmul_dev(self.h, t.h, act, _p(x_dev), _p(bias_dev), _p(y_dev), M), "bgl_matmul_dev")

    def matmul_group(self, ts, x_dev, ys, act=ACT_F32, biases=None):
        n = len(ts)
        M = 1 if x_dev.dim() == 1 else x_dev.shape[0]
        W = (C.c_void_p * n)(*[t.h.value for t in ts])
        Y = (C.c_void_p * n)(*[y.data_ptr() for y in ys])
        B = (C.c_void_p * n)(*[(b.data_ptr() if b is not None else None) for b in (biases or [None] * n)])
        _check(lib().bgl_matmul_group_dev(self.h, n, W, act, _p(x_dev), B, Y, M), "bgl_matmul_group_dev")

    def mlp(self, gate, up, down, x_dev, y_dev, act=ACT_F32, h_dev=None):
        """y = W_down (silu(W_gate x) * (W_up x)) on the device (bgl_mlp_dev); h_dev receives h."""
        M = 1 if x_dev.dim() == 1 else x_dev.shape[0]
        _check(lib().bgl_mlp_dev(self.h, gate.h, up.h, down.h, act, _p(x_dev), _p(y_dev), M, _p(h_dev)), "bgl_mlp_dev")

    def read_probe(self, ts, nblocks=0, nthreads=0):
        """Plain streaming read of the tensors' device bytes (the memory floor for a call)."""
        W = (C.c_void_p * len(ts))(*[t.h.value for t in ts])
        _check(lib().bgl_read_probe_dev(self.h, len(ts), W, nblocks, nthreads), "bgl_read_probe_dev")

    def prep_only(self, x_dev, act, t):
        """Prepare activation operands for tensor t's kind (kept in the context)."""
        M = 1 if x_dev.dim() == 1 else x_dev.shape[0]
        _check(lib().bgl_prep_act_dev(self.h, act, t.info()["kind"], _p(x_dev), M, x_dev.shape[-1]), "bgl_prep_act_dev")

    def matmul_prepped(self, t, y_dev, act=ACT_F32, bias_dev=None, M=1):
        _check(lib().bgl_matmul_prepped_dev(self.h, t.h, act, _p(bias_dev), _p(y_dev), M), "bgl_matmul_prepped_dev")

    def quant_act_i8(self, x_dev, gsize, xq_dev, ascale_dev):
        M = 1 if x_dev.dim() == 1 else x_dev.shape[0]
        _check(lib().bgl_quant_act_i8_dev(self.h, _p(x_dev), M, x_dev.shape[-1], gsize, _p(xq_dev), _p(ascale_dev)),
               "bgl_quant_act_i8_dev")

    # ---- int8 with one scale per token and per output channel ----
    def matmul_i8(self, ts, xq_dev, ascale_dev, ys, biases=None):
        """ys[i] = (codes xq [M][>= in] times the K_Q8C tensor ts[i]) * scales + biases[i] (bgl_matmul_i8_dev); ys are fp32,
        fp16 or bf16 tensors [M][out] of one type, whose rows may be apart.  A single tensor, y and bias need no lists."""
        if isinstance(ts, Tensor):
            ts, ys, biases = (ts,), (ys,), (biases,)
        f32, f16, bf16, i8 = _dtypes()
        n, dev = len(ts), self.device
        if not biases:
            biases = (None,) * n
        if not (0 < n == len(ys) == len(biases) and xq_dev.ndim == 2):
            _refuse("matmul_i8: one y (and bias) a tensor, codes [M][>= in]")
        M, width = xq_dev.shape
        ldq, dense = xq_dev.stride()
        inn, kind = ts[0].shape()[1], ys[0].dtype
        if xq_dev.dtype is not i8 or dense != 1 or width < inn:
            _refuse(f"matmul_i8: codes are dense int8 rows of at least in={inn}")
        # the kernels read the row's bytes up to the next multiple of 16
        if width < inn + 15 & -16 and xq_dev.storage_offset() + (M - 1) * ldq + (inn + 15 & -16) > xq_dev.untyped_storage().nbytes():
            _refuse("matmul_i8: the last row of codes ends before a multiple of 16 bytes")
        if ascale_dev.dtype is not f32 or ascale_dev.numel() != M or not ascale_dev.is_contiguous():
            _refuse(f"matmul_i8: scales are fp32 [{M}]")
        here = xq_dev.get_device() == dev == ascale_dev.get_device()
        W, Y, B, S = _arrays(n)
        for i in range(n):
            t, y, b = ts[i], ys[i], biases[i]
            out = t.shape()[0]
            if y.dtype is not kind or y.shape != (M, out):
                _refuse(f"matmul_i8: y is [{M}][{out}] of one type")
            ld, dense = y.stride()
            if dense != 1 and out > 1:
                _refuse("matmul_i8: rows of y are dense")
            here = here and y.get_device() == dev
            if b is not None:
                if b.dtype is not f32 or b.numel() != out or not b.is_contiguous():
                    _refuse(f"matmul_i8: a bias is fp32 [{out}]")
                here = here and b.get_device() == dev
                B[i] = b.data_ptr()
            W[i], Y[i], S[i] = t.h.value, y.data_ptr(), ld if M > 1 else out
        type_ = T_F32 if kind is f32 else T_F16 if kind is f16 else T_BF16 if kind is bf16 else _refuse("matmul_i8: y is fp32, fp16 or bf16")
        if not here:
            _refuse(f"matmul_i8: tensors lie on device {dev}")
        _check(lib().bgl_matmul_i8_dev(self.h, n, W, xq_dev.data_ptr(), ldq if M > 1 else width, ascale_dev.data_ptr(), B, Y, type_, S, M),
               "bgl_matmul_i8_dev")

    def norm(self, x, y=None, *, yq=None, yscale=None, kind=NORM_RMS, w=None, b=None, eps=1e-6, w_add=0.0, x_out=None, branch=None,
             branch_kind=NORM_NONE, branch_w=None, branch_b=None, branch_eps=1e-6, gate=None, alpha=1.0):
        """x_out = x + alpha * gate * branch_kind(branch), and y / (yq, yscale) = kind(x_out) (bgl_norm_dev) over [T][H] rows.
        gate: of the branch's type, [1][H], [T][1] or [T][H].  yq: int8 [T][H up to a multiple of 16], yscale: fp32 [T]."""
        T, H = x.shape
        dev = self.device
        d = capi.bgl_norm(T, H, *_rows(x, T, H, dev), _type(x))
        d.alpha, d.kind, d.eps = alpha, kind, eps
        if w_add:
            d.w_add = w_add
        if w is not None:
            d.w = _vec(w, H, dev)
        if b is not None:
            d.b = _vec(b, H, dev)
        if branch is not None:
            (d.f, d.ldf), d.f_type = _rows(branch, T, H, dev), _type(branch)
        if branch_kind:
            d.post, d.post_eps, d.post_w, d.post_b = branch_kind, branch_eps, _vec(branch_w, H, dev), _vec(branch_b, H, dev)
        if gate is not None:
            assert branch is not None and gate.dtype == branch.dtype and gate.dim() == 2
            assert gate.shape[0] in (1, T) and gate.shape[1] in (1, H) and (gate.shape[1] == 1 or gate.stride(1) == 1)
            if gate.get_device() != dev:
                _refuse(f"norm: tensors lie on device {dev}")
            d.gate, d.gate_t, d.gate_c = gate.data_ptr(), gate.stride(0) if gate.shape[0] > 1 else 0, int(gate.shape[1] > 1)
        if x_out is not None:
            assert x_out.dtype == x.dtype
            d.x_out, d.ldo = _rows(x_out, T, H, dev)
        if y is not None:
            (d.y, d.ldy), d.y_type = _rows(y, T, H, dev), _type(y)
        if yq is not None:
            rows, width = yq.shape if yq.ndim == 2 else (0, 0)
            ld, one = yq.stride() if rows == T else (0, 0)
            if one != 1 or width < H + 15 & -16 or yq.dtype is not _dtypes()[3] or yscale is None or yscale.numel() != T:
                _refuse(f"norm: yq is int8 [{T}][H={H} up to a multiple of 16] with dense rows, yscale [{T}]")
            if yq.get_device() != dev:
                _refuse(f"norm: tensors lie on device {dev}")
            d.yq, d.ldq, d.yscale = yq.data_ptr(), ld if T > 1 else width, _vec(yscale, T, dev)
        _check(lib().bgl_norm_dev(self.h, C.byref(d)), "bgl_norm_dev")

    # ---- attention: heads, the paged cache in 4 bits, the rows that attend ----
    def _heads(self, who, q, k, v, q_out, k_out, norm, q_w, k_w, eps, w_add, rope, pos, rot):
        dev, first = self.device, k if q is None else q
        if first is None or first.ndim != 3 or (q is None) != (q_out is None) or (k is None and k_out is not None):
            _refuse(f"{who}: q with q_out, or k, as [T][heads][D]")
        T, nq, D = shape = first.shape
        kind = first.dtype
        nk, Q, QO, K, KO, V, out = 0, _NO_ROWS, _NO_ROWS, _NO_ROWS, _NO_ROWS, _NO_ROWS, kind
        if q is not None:
            out = q_out.dtype
            Q, QO = _heads(q, shape, kind, dev, who), _heads(q_out, shape, out, dev, who)
        else:
            nq = 0
        if k is not None:
            nk = k.shape[1] if k.ndim == 3 else 0
            shape = (T, nk, D)
            K = _heads(k, shape, kind, dev, who)
            if v is not None:
                V = _heads(v, shape, kind, dev, who)
            if k_out is not None:
                if q is None:
                    out = k_out.dtype
                KO = _heads(k_out, shape, out, dev, who)
        n_pos = size = 0
        table = at = qw = kw = None
        if rope is None:
            rot = ROT_NONE
        elif rot:
            if rope.ndim != 2 or pos is None:
                _refuse(f"{who}: rope is fp32 [positions][rot], with pos int32 [{T}]")
            n_pos, size = rope.shape
            table, at = _floats(rope, n_pos * size, dev, who), _ints(pos, T, dev, who)
        if norm:
            qw, kw = _floats(q_w, D, dev, who), _floats(k_w, D, dev, who)
        return capi.bgl_heads(T, D, nq, nk, Q[0], K[0], V[0], Q[1], Q[2], K[1], K[2], V[1], V[2], _row_type(kind, who), norm, qw, kw, eps, w_add,
                              rot, size, table, n_pos, at, QO[0], KO[0], QO[1], QO[2], KO[1], KO[2], _row_type(out, who))

    def heads(self, q, k, q_out, k_out, *, norm=NORM_NONE, q_w=None, k_w=None, eps=1e-6, w_add=0.0, rope=None, pos=None, rot=ROT_HALF):
        """q_out, k_out = rotation(norm(q)), rotation(norm(k)) head by head (bgl_heads_dev) over [T][heads][D] tensors, whose tokens and
        heads may be apart; either pair may be None.  rope: fp32 [positions][rot] (cosines, then sines), pos: int32 [T]; rope
        None: no rotation."""
        d = self._heads("heads", q, k, None, q_out, k_out, norm, q_w, k_w, eps, w_add, rope, pos, rot)
        _check(lib().bgl_heads_dev(self.h, C.byref(d)), "bgl_heads_dev")

    def kv_append(self, cache, slots, k, v, *, q=None, q_out=None, norm=NORM_NONE, q_w=None, k_w=None, eps=1e-6, w_add=0.0, rope=None,
                  pos=None, rot=ROT_HALF):
        """Keys (normed and rotated as by heads) and values [T][heads][D] into the cache at slots int32 [T] (bgl_kv_append_dev),
        with q and q_out the queries in the same call."""
        d = self._heads("kv_append", q, k, v, q_out, None, norm, q_w, k_w, eps, w_add, rope, pos, rot)
        if cache.device != self.device:
            _refuse(f"kv_append: tensors lie on device {self.device}")
        _check(lib().bgl_kv_append_dev(self.h, C.byref(cache.d), C.byref(d), _ints(slots, d.T, self.device, "kv_append")), "bgl_kv_append_dev")

    def kv_read(self, cache, slots, k=None, v=None):
        """The values of the cache at slots int32 [n] into k and v [n][heads][D] (bgl_kv_read_dev); rows of slots outside the
        cache are left as they are."""
        one, n, dev = v if k is None else k, slots.numel(), self.device
        if one is None or cache.device != dev:
            _refuse(f"kv_read: k or v, and the cache, on device {dev}")
        shape, kind = (n, cache.heads, cache.dim), one.dtype
        K = _NO_ROWS if k is None else _heads(k, shape, kind, dev, "kv_read")
        V = _NO_ROWS if v is None else _heads(v, shape, kind, dev, "kv_read")
        _check(lib().bgl_kv_read_dev(self.h, C.byref(cache.d), _ints(slots, n, dev, "kv_read"), n, *K, *V, _row_type(kind, "kv_read")),
               "bgl_kv_read_dev")

    def attention(self, cache, q, out, start, lens, table, *, scale=None, causal=True, window=0, sink=None, max_rows=None, max_len=None):
        """out = attention of the rows q [T][heads][D] over the cache (bgl_attn_dev): sequence s has the rows start[s] ..
        start[s + 1] - 1 and lens[s] keys in the pages table[s]; int32 tensors [S + 1], [S], [S][pages].  scale None: 1 / sqrt(D).
        sink: fp32 [heads].  max_rows, max_len: the most rows and keys of a sequence, where the program knows them (None: as if every
        sequence had a row, and as many keys as the table's pages hold); kernels and launch shapes go by them, and so the order of
        sums, but no result needs them to be right."""
        dev, who = self.device, "attention"
        if table.ndim != 2 or q.ndim != 3 or q.shape[2] != cache.dim or cache.device != dev:
            _refuse(f"attention: q [T][heads][{cache.dim}], table [S][pages], the cache on device {dev}")
        S, ldt = table.shape
        T, nq, D = shape = q.shape
        kind = q.dtype
        a = capi.bgl_attn(S, T, nq, *_heads(q, shape, kind, dev, who), *_heads(out, shape, kind, dev, who), _row_type(kind, who),
                          _ints(start, S + 1, dev, who), _ints(lens, S, dev, who), _ints(table, S * ldt, dev, who), ldt,
                          D ** -0.5 if scale is None else scale, causal, window, _floats(sink, nq, dev, who),
                          max(1, T - S + 1) if max_rows is None else max_rows, ldt * cache.page if max_len is None else max_len)
        _check(lib().bgl_attn_dev(self.h, C.byref(cache.d), C.byref(a)), "bgl_attn_dev")

    # ---- MoE ----
    def bind_experts(self, descs):
        """descs: list of (kind, bits, packed, scales[, bias]) tuples, one per expert, of what bind takes; packed is
        2-D [out][row bytes or elements]; scales None for the dense kinds."""
        E = len(descs)
        arr = (capi.bgl_wt * E)()
        for e, d in enumerate(descs):
            kind, bits, pk, sc = d[:4]
            bi = d[4] if len(d) > 4 else None
            out = pk.shape[0]
            if kind in (K_F16, K_F32):
                inn = pk.shape[1]
            elif kind == K_MXFP4:                # GGUF blocks of 32 values, 17 bytes each
                inn = pk.reshape(out, -1).shape[1] // 17 * 32
            elif kind == K_Q8C:
                inn = pk.shape[1]
            else:
                inn = sc.shape[1] * (32 if kind == K_Q4G32H else 64)
            b = bits if kind == K_QNG64 else (8 if kind in (K_Q8G64, K_Q8C) else 4)
            _weights(kind, out, inn, pk, sc, bi)
            arr[e] = capi.bgl_wt(kind, b, out, inn, _w(pk), _w(sc), _w(bi))
        h = C.c_void_p()
        _check(lib().bgl_bind_experts(self.h, E, arr, C.byref(h)), "bgl_bind_experts")
        return Tensor(h)

    def experts_from_tensors(self, tensors):
        """Stack bound single tensors (e.g. from quantize()) into one expert tensor.  The new
        tensor owns them: their handles are cleared here and freed with the stack."""
        E = len(tensors)
        arr = (C.c_void_p * E)(*[t.h.value for t in tensors])
        h = C.c_void_p()
        _check(lib().bgl_experts_from_tensors(self.h, E, arr, C.byref(h)), "bgl_experts_from_tensors")
        for t in tensors:
            t.h = None
        return Tensor(h)

    def gather_matvec(self, experts, x_dev, idx_dev, y_dev):
        _check(lib().bgl_gather_matvec_dev(self.h, experts.h, _p(x_dev), _p(idx_dev), x_dev.shape[0], _p(y_dev)),
               "bgl_gather_matvec_dev")

    def moe_ffn(self, gate, up, down, shared, x_dev, idx_dev, w_dev, out_dev):
        sg, su, sd = (shared or (None, None, None))
        T, K = idx_dev.shape
        _check(lib().bgl_moe_ffn_dev(self.h, gate.h, up.h, down.h, sg.h if sg else None, su.h if su else None,
                                     sd.h if sd else None, _p(x_dev), _p(idx_dev), _p(w_dev), T, K, _p(out_dev)),
               "bgl_moe_ffn_dev")

    def moe_route(self, router_w, x_dev, K, idx_dev, w_dev, router_b=None, renorm=False):
        E, inn = router_w.shape
        _check(lib().bgl_moe_route_dev(self.h, _p(router_w), _p(router_b) if router_b is not None else None, E, inn, _p(x_dev),
                                       x_dev.shape[0], K, 1 if renorm else 0, _p(idx_dev), _p(w_dev)), "bgl_moe_route_dev")

    def moe_layer(self, router_w, gate, up, down, shared, x_dev, K, out_dev, router_b=None, renorm=False):
        sg, su, sd = (shared or (None, None, None))
        _check(lib().bgl_moe_layer_dev(self.h, _p(router_w), _p(router_b) if router_b is not None else None, 1 if renorm else 0,
                                       gate.h, up.h, down.h, sg.h if sg else None, su.h if su else None, sd.h if sd else None,
                                       _p(x_dev), x_dev.shape[0], K, _p(out_dev)), "bgl_moe_layer_dev")


class Model:
    """Weights loaded from the int4 layout manifest + blob (bgl_model_load_int4) or from the
    repacked-layout cache (bgl_model_load_cache)."""

    def __init__(self, ctx, layout, blob, cache=None):
        self.ctx, self.layout, self.blob = ctx, layout, blob
        h = C.c_void_p()
        if cache is not None:
            _check(lib().bgl_model_load_cache(ctx.h, cache.encode(), layout.encode(), blob.encode(), C.byref(h)),
                   "bgl_model_load_cache")
        else:
            _check(lib().bgl_model_load_int4(ctx.h, layout.encode(), blob.encode(), C.byref(h)), "bgl_model_load_int4")
        self.h = h

    def __len__(self):
        return lib().bgl_model_count(self.h)

    def find(self, name):
        """(kind, out, in, Tensor or None, address of the f32 data or None); the model owns the tensor."""
        k, o, i = C.c_int(), C.c_int(), C.c_int()
        t, f = C.c_void_p(), C.c_void_p()
        _check(lib().bgl_model_find(self.h, name.encode(), C.byref(k), C.byref(o), C.byref(i), C.byref(t), C.byref(f)),
               "bgl_model_find")
        return k.value, o.value, i.value, (Tensor(t) if t.value else None), f.value

    def save_cache(self, path):
        _check(lib().bgl_model_save_cache(self.h, path.encode(), self.layout.encode(), self.blob.encode()), "bgl_model_save_cache")

    def close(self):
        if self.h:
            lib().bgl_model_free(self.h)
            self.h = None


def layout_check(layout, blob):
    n = C.c_int()
    rc = lib().bgl_int4_layout_check(layout.encode(), blob.encode(), C.byref(n))
    return rc, n.value


def af_layout_check(layout, blob_bytes):
    n = C.c_int()
    rc = lib().bgl_af_layout_check(layout.encode(), blob_bytes, C.byref(n))
    return rc, n.value


def cache_valid(cache, layout, blob):
    return lib().bgl_model_cache_valid(cache.encode(), layout.encode(), blob.encode())


# ---- the name-keyed registry (mlx_moe.h boundary): thin wrappers, 1 = ok / 0 = failure ----
class Registry:
    """bgl_gpu_* entry points with numpy host buffers."""

    @staticmethod
    def L():
        return lib()

    def available(self):
        return lib().bgl_gpu_available()

    def bind_af(self, blob, name, E, out, inn, ng, packed_off, scale_off, bias_off, bits):
        return lib().bgl_gpu_bind_af(blob.ctypes.data, blob.nbytes, name.encode(), E, out, inn, ng, packed_off,
                                     scale_off, bias_off, bits)

    def load_layout_af(self, layout, blob):
        """Binds every tensor of an AF layout manifest over blob (uint8 array); the count or -1."""
        return lib().bgl_gpu_load_layout_af(layout.encode(), blob.ctypes.data, blob.nbytes)

    def binding_kind(self, name):
        b = C.c_int()
        k = lib().bgl_gpu_binding_kind(name.encode(), C.byref(b))
        return k, b.value

    def snapshot(self, name):
        sid = C.c_uint64()
        ok = lib().bgl_gpu_snapshot_binding(name.encode(), C.byref(sid))
        return ok, sid.value

    def dequant_probe(self, name, e, row, col0, ncols):
        import numpy as np
        out = np.zeros(ncols, np.float32)
        ok = lib().bgl_gpu_dequant_probe(name.encode(), e, row, col0, ncols, out.ctypes.data)
        return ok, out

    def matvec_probe(self, name, e, x, out):
        import numpy as np
        x = np.ascontiguousarray(x, np.float32)
        y = np.zeros(out, np.float32)
        ok = lib().bgl_gpu_matvec_probe(name.encode(), e, x.ctypes.data, y.ctypes.data)
        return ok, y

    def ffn_gather(self, name, x, idx, out):
        import numpy as np
        x = np.ascontiguousarray(x, np.float32)
        idx = np.ascontiguousarray(idx, np.int32)
        y = np.zeros((x.shape[0], out), np.float32)
        ok = lib().bgl_gpu_ffn_gather(name.encode(), x.ctypes.data, x.shape[0], idx.ctypes.data, y.ctypes.data)
        return ok, y

    def bind_mixed(self, name, planes, offsets, bits, scales, out, inn):
        return lib().bgl_gpu_bind_qng64_mixed_dense_probe(planes.ctypes.data, planes.nbytes, offsets.ctypes.data,
                                                          bits.ctypes.data, scales.ctypes.data, name.encode(), out, inn)

    def mixed_probe(self, planes, offsets, bits, scales, out, inn, x):
        import numpy as np
        x = np.ascontiguousarray(x, np.float32)
        y = np.zeros((x.shape[0], out), np.float32)
        ok = lib().bgl_gpu_qng64_mixed_dense_probe(planes.ctypes.data, planes.nbytes, offsets.ctypes.data, bits.ctypes.data,
                                                   scales.ctypes.data, out, inn, x.ctypes.data, x.shape[0], y.ctypes.data)
        return ok, y

    def bind_router(self, name, w, bias=None):
        import numpy as np
        w = np.ascontiguousarray(w, np.float32)
        b = np.ascontiguousarray(bias, np.float32) if bias is not None else None
        return lib().bgl_gpu_bind_router(name.encode(), w.ctypes.data, b.ctypes.data if b is not None else None,
                                         w.shape[0], w.shape[1])

    def moe_layer(self, router, gate, up, down, shared, x, K, renorm=False):
        import numpy as np
        x = np.ascontiguousarray(x, np.float32)
        out = np.zeros_like(x)
        idx = np.zeros((x.shape[0], K), np.int32)
        w = np.zeros((x.shape[0], K), np.float32)
        sg, su, sd = [s.encode() if s else None for s in (shared or (None, None, None))]
        ok = lib().bgl_gpu_moe_layer(router.encode(), gate.encode(), up.encode(), down.encode(), sg, su, sd, x.ctypes.data,
                                     x.shape[0], K, 1 if renorm else 0, out.ctypes.data, idx.ctypes.data, w.ctypes.data)
        return ok, out, idx, w

    def moe_ffn(self, gate, up, down, shared, x, idx, w):
        import numpy as np
        x = np.ascontiguousarray(x, np.float32)
        idx = np.ascontiguousarray(idx, np.int32)
        w = np.ascontiguousarray(w, np.float32)
        out = np.zeros_like(x)
        sg, su, sd = [s.encode() if s else None for s in (shared or (None, None, None))]
        ok = lib().bgl_gpu_moe_ffn(gate.encode(), up.encode(), down.encode(), sg, su, sd, x.ctypes.data, x.shape[0],
                                   idx.ctypes.data, w.ctypes.data, idx.shape[1], out.ctypes.data)
        return ok, out
