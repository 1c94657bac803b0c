// bgl_norm.hip -- the end of a transformer block and the norm before the next one, in one launch
// (forward_token's residual adds and rmsnorm, qwen_infer.c:1435-1585, with the norm after the block, the
// gate and the residual scale that other models put there):
//
//   n = post(f)                              f: the block's output (or none)
//   v = x + alpha * gate * n                 rounded once to x's type: the new residual row
//   y = pre(v)                               as floats, or as int8 codes with one scale per token
//
//   rms(v)   = v / sqrt(mean(v^2) + eps) * (w + w_add)
//   layer(v) = (v - mean(v)) / sqrt(mean((v - mean)^2) + eps) * (w + w_add) + b
//
// Every value is computed in double and rounded once to fp32 (and from there to a 16-bit type): a code
// of the int8 output changes by one where a value lies within rounding of a border between codes, and
// with the values right to fp32's last bit the codes are those of the formula.  gfx950 issues double
// multiply-adds at the rate of single ones, and the launch is bound by memory.
//
// The row stays in registers between its two passes (statistics, then the output): 16 values a thread,
// 64 threads to a row up to H = 1024, 256 up to 4096, 1024 up to 16384.  Wider rows (the quantizer takes
// MLP rows) go through k_norm_wide, which reads the row again for each pass.  A workgroup walks several
// rows, so the norm weights are read once per workgroup and kept.
#include <string.h>

#include <algorithm>

#include "../../include/beglin_qgemv.h"
#include "bgl_i8.h"

#define HIPCHK(expr)                                                                             \
    do {                                                                                         \
        hipError_t e_ = (expr);                                                                  \
        if (e_ != hipSuccess) return bgl_fail(BGL_E_HIP, "%s: %s", #expr, hipGetErrorString(e_)); \
    } while (0)

struct NormLaunch {
    bgl_norm d;
    const float *glu_u;      // x is an MLP block's gate row: v = silu(x) * u, which goes to x_out (bgl_mlp.hip's h)
};

#define NORM_V 8             // consecutive values of a thread
#define NORM_NV 2            // such runs

template <bool VEC>
__device__ __forceinline__ void norm_ld8(float (&o)[NORM_V], const void *p, int type, size_t at, int left) {
    if constexpr (VEC) {
        if (left <= 0) {
#pragma unroll
            for (int j = 0; j < NORM_V; j++) o[j] = 0.0f;
        } else if (type == BGL_T_F32) {
            const i8_f4 *q = (const i8_f4 *)((const float *)p + at);
            const i8_f4 a = q[0], b = q[1];
#pragma unroll
            for (int j = 0; j < 4; j++) { o[j] = a[j]; o[4 + j] = b[j]; }
        } else {
            const i8_u4 a = *(const i8_u4 *)((const uint16_t *)p + at);
#pragma unroll
            for (int j = 0; j < NORM_V; j++) {
                const uint16_t h = (uint16_t)(a[j / 2] >> (16 * (j & 1)));
                o[j] = type == BGL_T_F16 ? (float)__builtin_bit_cast(_Float16, h) : __uint_as_float((uint32_t)h << 16);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < NORM_V; j++) o[j] = j < left ? i8_ld(p, type, at + j) : 0.0f;
    }
}

template <bool VEC>
__device__ __forceinline__ void norm_st8(void *p, int type, size_t at, int left, const float (&v)[NORM_V]) {
    if constexpr (VEC) {
        if (left <= 0) return;
        if (type == BGL_T_F32) {
            i8_f4 *q = (i8_f4 *)((float *)p + at);
            q[0] = i8_f4{v[0], v[1], v[2], v[3]};
            q[1] = i8_f4{v[4], v[5], v[6], v[7]};
        } else {
            i8_u4 a;
#pragma unroll
            for (int j = 0; j < 4; j++) a[j] = (uint32_t)i8_h16(v[2 * j], type) | ((uint32_t)i8_h16(v[2 * j + 1], type) << 16);
            *(i8_u4 *)((uint16_t *)p + at) = a;
        }
    } else {
#pragma unroll
        for (int j = 0; j < NORM_V; j++)
            if (j < left) i8_st(p, type, at + j, v[j]);
    }
}

// Sums over the NT threads of a row, in every one of them, in one order whatever the launch.
template <int NT>
__device__ __forceinline__ double row_sum(double v, double *red) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    if constexpr (NT > 64) {
        const int wave = threadIdx.x >> 6;
        __syncthreads();                       // the last round's reads are done
        if ((threadIdx.x & 63) == 0) red[wave] = v;
        __syncthreads();
        v = 0.0;
#pragma unroll
        for (int i = 0; i < NT / 64; i++) v += red[i];
    }
    return v;
}
template <int NT>
__device__ __forceinline__ uint32_t row_max(uint32_t v, double *red) {
    v = wave_max_u32(v);
    if constexpr (NT > 64) {
        uint32_t *r = (uint32_t *)red;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NT / 64; i++) v = max(v, r[i]);
    }
    return v;
}

// mean and 1 / sqrt(... + eps) of a norm over the thread's values (0 past the row's end)
template <int NT, int NVAL>
__device__ __forceinline__ void norm_stats(int kind, const float (&v)[NVAL], const bool (&in)[NVAL], int H, float eps, double *red,
                                           double &mean, double &inv) {
    mean = 0.0;
    if (kind == BGL_NORM_LAYER) {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < NVAL; i++) s += (double)v[i];
        mean = row_sum<NT>(s, red) / H;
    }
    double q = 0.0;
#pragma unroll
    for (int i = 0; i < NVAL; i++) {
        const double d = in[i] ? (double)v[i] - mean : 0.0;
        q = fma(d, d, q);
    }
    inv = 1.0 / sqrt(row_sum<NT>(q, red) / H + (double)eps);
}

template <int NT, bool VEC>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void k_norm(NormLaunch L) {
    constexpr int RPW = NT < 256 ? 256 / NT : 1, NVAL = NORM_V * NORM_NV;
    const bgl_norm &d = L.d;
    __shared__ double red[16];
    const int lt = NT < 256 ? threadIdx.x % NT : threadIdx.x;
    int at[NORM_NV], left[NORM_NV];
    bool in[NVAL];
#pragma unroll
    for (int i = 0; i < NORM_NV; i++) {
        at[i] = (i * NT + lt) * NORM_V;
        left[i] = d.H - at[i];
#pragma unroll
        for (int j = 0; j < NORM_V; j++) in[i * NORM_V + j] = j < left[i];
    }
    // the weights of the norm before the next block stay for every row of the workgroup
    float w[NVAL];
#pragma unroll
    for (int i = 0; i < NVAL; i++) w[i] = 1.0f;
    if (d.w) {
#pragma unroll
        for (int i = 0; i < NORM_NV; i++)
            norm_ld8<VEC>(*(float(*)[NORM_V])(w + i * NORM_V), d.w, BGL_T_F32, at[i], left[i]);
    }
    for (long row = (long)blockIdx.x * RPW + (NT < 256 ? threadIdx.x / NT : 0); row < d.T; row += (long)gridDim.x * RPW) {
        float v[NVAL];
#pragma unroll
        for (int i = 0; i < NORM_NV; i++)
            norm_ld8<VEC>(*(float(*)[NORM_V])(v + i * NORM_V), d.x, d.x_type, (size_t)row * d.ldx + at[i], left[i]);
        if (L.glu_u) {
            float u[NVAL];
#pragma unroll
            for (int i = 0; i < NORM_NV; i++)
                norm_ld8<VEC>(*(float(*)[NORM_V])(u + i * NORM_V), L.glu_u, BGL_T_F32, (size_t)row * d.ldx + at[i], left[i]);
#pragma unroll
            for (int k = 0; k < NVAL; k++) v[k] = in[k] ? i8_swiglu(v[k], u[k]) : 0.0f;
        }
        if (d.f) {
            float f[NVAL], g[NVAL];
#pragma unroll
            for (int i = 0; i < NORM_NV; i++)
                norm_ld8<VEC>(*(float(*)[NORM_V])(f + i * NORM_V), d.f, d.f_type, (size_t)row * d.ldf + at[i], left[i]);
            if (d.gate) {
                if (d.gate_c) {
#pragma unroll
                    for (int i = 0; i < NORM_NV; i++)
                        norm_ld8<VEC>(*(float(*)[NORM_V])(g + i * NORM_V), d.gate, d.f_type, (size_t)row * d.gate_t + at[i], left[i]);
                } else {
                    const float g1 = i8_ld(d.gate, d.f_type, (size_t)row * d.gate_t);
#pragma unroll
                    for (int i = 0; i < NVAL; i++) g[i] = g1;
                }
            }
            double mean = 0.0, inv = 1.0;
            if (d.post != BGL_NORM_NONE) norm_stats<NT, NVAL>(d.post, f, in, d.H, d.post_eps, red, mean, inv);
#pragma unroll
            for (int i = 0; i < NORM_NV; i++) {
                float pw[NORM_V], pb[NORM_V];
                if (d.post != BGL_NORM_NONE && d.post_w) norm_ld8<VEC>(pw, d.post_w, BGL_T_F32, at[i], left[i]);
                if (d.post != BGL_NORM_NONE && d.post_b) norm_ld8<VEC>(pb, d.post_b, BGL_T_F32, at[i], left[i]);
#pragma unroll
                for (int j = 0; j < NORM_V; j++) {
                    const int k = i * NORM_V + j;
                    double n = (double)f[k];
                    if (d.post != BGL_NORM_NONE) {
                        n = (n - mean) * inv;
                        if (d.post_w) n *= (double)pw[j] + (double)d.w_add;
                        if (d.post_b) n += (double)pb[j];
                    }
                    if (d.gate) n *= (double)g[k];
                    v[k] = in[k] ? i8_kept((float)((double)v[k] + (double)d.alpha * n), d.x_type) : 0.0f;
                }
            }
        }
        if (d.x_out) {
#pragma unroll
            for (int i = 0; i < NORM_NV; i++)
                norm_st8<VEC>(d.x_out, d.x_type, (size_t)row * d.ldo + at[i], left[i], *(float(*)[NORM_V])(v + i * NORM_V));
        }
        if (!d.y && !d.yq) continue;
        if (d.kind != BGL_NORM_NONE) {
            double mean, inv;
            norm_stats<NT, NVAL>(d.kind, v, in, d.H, d.eps, red, mean, inv);
#pragma unroll
            for (int i = 0; i < NORM_NV; i++) {
                float b[NORM_V];
                if (d.b) norm_ld8<VEC>(b, d.b, BGL_T_F32, at[i], left[i]);
#pragma unroll
                for (int j = 0; j < NORM_V; j++) {
                    const int k = i * NORM_V + j;
                    double n = ((double)v[k] - mean) * inv;
                    if (d.w) n *= (double)w[k] + (double)d.w_add;
                    if (d.b) n += (double)b[j];
                    v[k] = (float)n;
                }
            }
        }
        if (d.y) {
#pragma unroll
            for (int i = 0; i < NORM_NV; i++)
                norm_st8<VEC>(d.y, d.y_type, (size_t)row * d.ldy + at[i], left[i], *(float(*)[NORM_V])(v + i * NORM_V));
        }
        if (d.yq) {
            uint32_t mb = I8_MX0;
#pragma unroll
            for (int k = 0; k < NVAL; k++)
                if (in[k]) mb = max(mb, __float_as_uint(v[k]) & 0x7fffffffu);
            const I8Scale s = i8_scale(row_max<NT>(mb, red));
            if (lt == 0) d.yscale[row] = s.sc;
            int8_t *q = d.yq + (size_t)row * d.ldq;
#pragma unroll
            for (int i = 0; i < NORM_NV; i++) {
                uint32_t c2[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float *t = v + i * NORM_V + 4 * j;
                    const bool *u = in + i * NORM_V + 4 * j;
                    c2[j] = i8_pack4(u[0] ? i8_code(t[0], s) : 0, u[1] ? i8_code(t[1], s) : 0, u[2] ? i8_code(t[2], s) : 0,
                                     u[3] ? i8_code(t[3], s) : 0);
                }
                // rows are 16 bytes apart at least: whole runs of 8, the bytes up to the row's next multiple of 16 zeroed
                if (at[i] < ((d.H + 15) & ~15)) *(uint2 *)(q + at[i]) = make_uint2(c2[0], c2[1]);
            }
        }
    }
}

// Rows wider than 16384: 1024 threads a row, one value at a time, the row read again for each pass.
// Only the thread that wrote a value of x_out reads it back.
__global__ __launch_bounds__(1024) void k_norm_wide(NormLaunch L) {
    const bgl_norm &d = L.d;
    __shared__ double red[16];
    const int tid = threadIdx.x;
    for (long row = blockIdx.x; row < d.T; row += gridDim.x) {
        double fmean = 0.0, finv = 1.0;
        if (d.f && d.post != BGL_NORM_NONE) {
            if (d.post == BGL_NORM_LAYER) {
                double s = 0.0;
                for (int h = tid; h < d.H; h += 1024) s += (double)i8_ld(d.f, d.f_type, (size_t)row * d.ldf + h);
                fmean = row_sum<1024>(s, red) / d.H;
            }
            double q = 0.0;
            for (int h = tid; h < d.H; h += 1024) {
                const double t = (double)i8_ld(d.f, d.f_type, (size_t)row * d.ldf + h) - fmean;
                q = fma(t, t, q);
            }
            finv = 1.0 / sqrt(row_sum<1024>(q, red) / d.H + (double)d.post_eps);
        }
        auto fresh = [&](int h) -> float {               // the new residual value
            float v = i8_ld(d.x, d.x_type, (size_t)row * d.ldx + h);
            if (L.glu_u) v = i8_swiglu(v, L.glu_u[(size_t)row * d.ldx + h]);
            if (!d.f) return v;
            double n = (double)i8_ld(d.f, d.f_type, (size_t)row * d.ldf + h);
            if (d.post != BGL_NORM_NONE) {
                n = (n - fmean) * finv;
                if (d.post_w) n *= (double)d.post_w[h] + (double)d.w_add;
                if (d.post_b) n += (double)d.post_b[h];
            }
            if (d.gate) n *= (double)i8_ld(d.gate, d.f_type, (size_t)row * d.gate_t + (d.gate_c ? h : 0));
            return i8_kept((float)((double)v + (double)d.alpha * n), d.x_type);
        };
        if (d.x_out)
            for (int h = tid; h < d.H; h += 1024) i8_st(d.x_out, d.x_type, (size_t)row * d.ldo + h, fresh(h));
        // x_out may be x itself: from here on its new values are read
        auto value = [&](int h) -> float { return d.x_out ? i8_ld(d.x_out, d.x_type, (size_t)row * d.ldo + h) : fresh(h); };
        if (!d.y && !d.yq) continue;
        double mean = 0.0, inv = 1.0;
        if (d.kind == BGL_NORM_LAYER) {
            double s = 0.0;
            for (int h = tid; h < d.H; h += 1024) s += (double)value(h);
            mean = row_sum<1024>(s, red) / d.H;
        }
        if (d.kind != BGL_NORM_NONE) {
            double q = 0.0;
            for (int h = tid; h < d.H; h += 1024) {
                const double t = (double)value(h) - mean;
                q = fma(t, t, q);
            }
            inv = 1.0 / sqrt(row_sum<1024>(q, red) / d.H + (double)d.eps);
        }
        auto out = [&](int h) -> float {
            const float v = value(h);
            if (d.kind == BGL_NORM_NONE) return v;
            double n = ((double)v - mean) * inv;
            if (d.w) n *= (double)d.w[h] + (double)d.w_add;
            if (d.b) n += (double)d.b[h];
            return (float)n;
        };
        uint32_t mb = I8_MX0;
        for (int h = tid; h < d.H; h += 1024) {
            const float v = out(h);
            if (d.y) i8_st(d.y, d.y_type, (size_t)row * d.ldy + h, v);
            mb = max(mb, __float_as_uint(v) & 0x7fffffffu);
        }
        if (!d.yq) continue;
        const I8Scale s = i8_scale(row_max<1024>(mb, red));
        if (tid == 0) d.yscale[row] = s.sc;
        int8_t *q = d.yq + (size_t)row * d.ldq;
        for (int h = tid; h < ((d.H + 15) & ~15); h += 1024) q[h] = (int8_t)(h < d.H ? i8_code(out(h), s) : 0);
    }
}

// ================================================================================== host side
#define NORM_BLOCKS 2048         // workgroups of a launch at most (8 a CU): each then walks its rows

static int norm_launch(bgl_ctx *c, const NormLaunch &L, bool vec) {
    const bgl_norm &d = L.d;
    int tok = prof_begin(c, L.glu_u || d.kind == BGL_NORM_NONE ? 0 : 2);
    auto go = [&](auto kernel, int threads, int rows) {
        const long blocks = std::min<long>(NORM_BLOCKS, ((long)d.T + rows - 1) / rows);
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), 0, c->stream, L);
    };
    if (d.H <= 1024) vec ? go(k_norm<64, true>, 256, 4) : go(k_norm<64, false>, 256, 4);
    else if (d.H <= 4096) vec ? go(k_norm<256, true>, 256, 1) : go(k_norm<256, false>, 256, 1);
    else if (d.H <= 16384) vec ? go(k_norm<1024, true>, 1024, 1) : go(k_norm<1024, false>, 1024, 1);
    else go(k_norm_wide, 1024, 1);
    prof_end(c, tok);
    HIPCHK(hipGetLastError());
    return 0;
}

int run_quant_rows(bgl_ctx *c, const float *x, const float *u, float *h, int M, int K, int8_t *xq, long ldq, float *xs) {
    NormLaunch L;
    memset(&L, 0, sizeof L);
    L.d.T = M; L.d.H = K;
    L.d.x = x; L.d.ldx = K; L.d.x_type = BGL_T_F32;
    L.glu_u = u;
    L.d.x_out = u ? h : nullptr; L.d.ldo = K;
    L.d.yq = xq; L.d.ldq = ldq; L.d.yscale = xs;
    return norm_launch(c, L, K % 8 == 0 && (((uintptr_t)x | (uintptr_t)u | (uintptr_t)h) & 15) == 0);
}

extern "C" int bgl_norm_dev(bgl_ctx *c, const bgl_norm *d) {
    if (!c || !d || !d->x) return bgl_fail(BGL_E_ARG, "bgl_norm_dev: NULL argument");
    if (d->T < 1 || d->H < 1) return bgl_fail(BGL_E_ARG, "bgl_norm_dev: T=%d H=%d", d->T, d->H);
    auto type_ok = [](int t) { return t == BGL_T_F32 || t == BGL_T_F16 || t == BGL_T_BF16; };
    auto kind_ok = [](int k) { return k == BGL_NORM_NONE || k == BGL_NORM_RMS || k == BGL_NORM_LAYER; };
    if (!type_ok(d->x_type) || (d->f && !type_ok(d->f_type)) || (d->y && !type_ok(d->y_type)))
        return bgl_fail(BGL_E_ARG, "bgl_norm_dev: unknown element type");
    if (!kind_ok(d->kind) || !kind_ok(d->post)) return bgl_fail(BGL_E_ARG, "bgl_norm_dev: unknown norm kind");
    if (!d->f && (d->post != BGL_NORM_NONE || d->gate))
        return bgl_fail(BGL_E_ARG, "bgl_norm_dev: a norm after the block or a gate needs the block's output f");
    if (!d->x_out && !d->y && !d->yq) return bgl_fail(BGL_E_ARG, "bgl_norm_dev: nothing to write (x_out, y and yq are NULL)");
    if ((d->yq != nullptr) != (d->yscale != nullptr)) return bgl_fail(BGL_E_ARG, "bgl_norm_dev: yq and yscale go together");
    const long h = d->H;
    if (d->ldx < h || (d->f && d->ldf < h) || (d->x_out && d->ldo < h) || (d->y && d->ldy < h))
        return bgl_fail(BGL_E_ARG, "bgl_norm_dev: a row stride is below H=%d", d->H);
    if (d->gate && ((d->gate_c != 0 && d->gate_c != 1) || d->gate_t < 0 || (d->gate_c && d->gate_t && d->gate_t < h)))
        return bgl_fail(BGL_E_ARG, "bgl_norm_dev: gate strides %ld, %ld (channels 0 or 1; tokens 0, or at least H with channels)",
                        d->gate_t, d->gate_c);
    if (d->yq && (d->ldq < ((h + 15) & ~15l) || d->ldq % 16 || (uintptr_t)d->yq % 16))
        return bgl_fail(BGL_E_ARG, "bgl_norm_dev: code rows are 16-byte aligned, a multiple of 16 and at least H bytes apart (ldq=%ld)", d->ldq);
    if (d->x_out == d->x && d->ldo != d->ldx) return bgl_fail(BGL_E_ARG, "bgl_norm_dev: x_out is x with another row stride");
    if (d->y && (d->y == d->x || d->y == d->f || d->y == d->x_out || d->y == d->gate))
        return bgl_fail(BGL_E_ARG, "bgl_norm_dev: y is one of the other rows");
    if (d->f && (d->x_out == d->f || (d->gate && d->x_out == d->gate)))
        return bgl_fail(BGL_E_ARG, "bgl_norm_dev: x_out may be x, not f or the gate");
    HIPCHK(hipSetDevice(c->device));
    NormLaunch L;
    memset(&L, 0, sizeof L);
    L.d = *d;
    // 16-byte accesses where every row starts on 16 bytes and holds whole runs of 8 values
    auto al = [](const void *p, long ld, int type) { return !p || (((uintptr_t)p | (uintptr_t)ld * i8_elem(type)) & 15) == 0; };
    const bool vec = h % 8 == 0 && al(d->x, d->ldx, d->x_type) && al(d->f, d->ldf, d->f_type) && al(d->x_out, d->ldo, d->x_type) &&
                     al(d->y, d->ldy, d->y_type) && al(d->gate_c ? d->gate : nullptr, d->gate_t, d->f_type) &&
                     al(d->w, 0, BGL_T_F32) && al(d->b, 0, BGL_T_F32) && al(d->post_w, 0, BGL_T_F32) && al(d->post_b, 0, BGL_T_F32);
    return norm_launch(c, L, vec);
}
