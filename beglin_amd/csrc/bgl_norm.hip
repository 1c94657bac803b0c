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
// multiply-adds at the rate of single ones.  Rows normed once are bound by memory: 4096 rows of 4096 in bf16
// (residual add, RMS norm) take 31 us, 4.4 TB/s of what they read and write, where a large copy moves 5.1, and the
// vector units issue for 11 of them.  Rows normed twice are not: 777 of 2883 with two layer norms and a gate take 15.3 us,
// of which 7 to 9 are issue (77 instructions a value's place), 6 the bytes, and the waves wait 58% of the time, for loads
// and at the barriers of four sums.
//
// The row stays in registers between its passes (statistics, then the output): a wave to a row up to H = 512, then
// workgroups of 256, 512 or 1024 threads with 8 or 16 values each.  Wider
// rows (the quantizer takes MLP rows) go through k_norm_wide, which reads the row again for each pass.
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

// What a row is before the norm: itself, x + a gated block, x + a normed and gated block, or SwiGLU of two rows.
enum { ROW_X = 0, ROW_ADD = 1, ROW_POST = 2, ROW_GLU = 3 };

// 16 bytes of a row, wherever the row starts (gfx950 loads and stores them at any address)
typedef float nr_f4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned int nr_u4 __attribute__((ext_vector_type(4), aligned(2)));

// A thread's values of a row of at least 8: NV chunks of 8 consecutive ones, NT chunks apart.  A chunk that the row's
// end cuts, or that lies behind it, loads the row's last 8 values instead and shifts its own to the front (values past
// the end are 0 and stay so): every load is a full one and none is conditional.
// NT: threads of a row, or 0: as many as the workgroup has.
template <int NT, int NV>
struct RowMap {
    static constexpr int N = 8 * NV;
    int lt, H;
    __device__ __forceinline__ int at(int i) const { return (i * (NT ? NT : (int)blockDim.x) + lt) * 8; }
    __device__ __forceinline__ int has(int i) const { return H - at(i); }        // values of chunk i that exist (>= 8: all)
    // An access is a uniform address plus the thread's 32-bit offset: no address registers per pointer and value.
    template <typename V>
    __device__ __forceinline__ V get(const void *row, int i, int per, int j = 0) const {
        return *(const V *)((const char *)row + (uint32_t)(min(at(i), H - 8) + j) * (uint32_t)per);
    }
    template <typename V>
    __device__ __forceinline__ void put(void *row, int i, int per, V v, int j = 0) const {
        *(V *)((char *)row + (uint32_t)(at(i) + j) * (uint32_t)per) = v;
    }
    __device__ __forceinline__ void load(float *q, int i, const void *row, int type) const {
        if (type == BGL_T_F32) {
            const nr_f4 u = get<nr_f4>(row, i, 4), v = get<nr_f4>(row, i, 4, 4);
#pragma unroll
            for (int j = 0; j < 4; j++) { q[j] = u[j]; q[4 + j] = v[j]; }
        } else {
            const nr_u4 u = get<nr_u4>(row, i, 2);
            if (type == BGL_T_F16) {
#pragma unroll
                for (int j = 0; j < 8; j++) q[j] = (float)__builtin_bit_cast(_Float16, (uint16_t)(u[j / 2] >> (16 * (j & 1))));
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) q[j] = __uint_as_float(j & 1 ? u[j / 2] & 0xffff0000u : u[j / 2] << 16);
            }
        }
        const int s = 8 - has(i);
        if (s > 0) {
#pragma unroll
            for (int step = 4; step; step >>= 1) {
#pragma unroll
                for (int j = 0; j < 8; j++) q[j] = s & step ? (j + step < 8 ? q[j + step] : 0.0f) : q[j];
            }
#pragma unroll
            for (int j = 0; j < 8; j++) q[j] = s >= 8 ? 0.0f : q[j];
        }
    }
    // zeroes what a computation made of the values past the end
    __device__ __forceinline__ void cut(float *q, int i) const {
        const int n = has(i);
        if (n >= 8) return;
#pragma unroll
        for (int j = 0; j < 8; j++) q[j] = j < n ? q[j] : 0.0f;
    }
    // chunk i rounded to the type and stored; with KEEP, q becomes what was stored
    template <bool KEEP>
    __device__ __forceinline__ void store(void *row, int type, float *q, int i) const {
        const int n = has(i);
        if (type == BGL_T_F32) {
            if (!row) return;
            if (n >= 8) {
                put(row, i, 4, nr_f4{q[0], q[1], q[2], q[3]});
                put(row, i, 4, nr_f4{q[4], q[5], q[6], q[7]}, 4);
            } else if (n > 0) {
#pragma unroll
                for (int j = 0; j < 7; j++)
                    if (j < n) put(row, i, 4, q[j], j);
            }
            return;
        }
        uint16_t h[8];
        if (type == BGL_T_F16) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                h[j] = __builtin_bit_cast(uint16_t, (_Float16)q[j]);
                if (KEEP) q[j] = (float)__builtin_bit_cast(_Float16, h[j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                h[j] = __builtin_bit_cast(uint16_t, (__bf16)q[j]);
                if (KEEP) q[j] = __uint_as_float((uint32_t)h[j] << 16);
            }
        }
        if (!row) return;
        if (n >= 8) {
            nr_u4 u;
#pragma unroll
            for (int j = 0; j < 4; j++) u[j] = (uint32_t)h[2 * j] | ((uint32_t)h[2 * j + 1] << 16);
            put(row, i, 2, u);
        } else if (n > 0) {
#pragma unroll
            for (int j = 0; j < 7; j++)
                if (j < n) put(row, i, 2, h[j], j);
        }
    }
};
// row `row` of rows ld values of a type apart
__device__ __forceinline__ const void *norm_row(const void *p, long row, long ld, int type) { return (const char *)p + row * ld * (type == BGL_T_F32 ? 4 : 2); }

// n = (v - mean) * inv * (w + w_add) + b of a chunk, for any of its parts (the conditions are the launch's, outside the
// loops over values)
template <typename Map>
__device__ __forceinline__ void norm_chunk(double (&n)[8], const Map &m, int i, const float *v, int kind, double mean, double inv, const float *w,
                                           float w_add, const float *b) {
    float p[8];
    if (kind == BGL_NORM_LAYER) {
#pragma unroll
        for (int j = 0; j < 8; j++) n[j] = ((double)v[j] - mean) * inv;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) n[j] = (double)v[j] * inv;
    }
    if (w) {
        m.load(p, i, w, BGL_T_F32);
        if (w_add == 0.0f) {
#pragma unroll
            for (int j = 0; j < 8; j++) n[j] *= (double)p[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) n[j] *= (double)p[j] + (double)w_add;
        }
    }
    if (b) {
        m.load(p, i, b, BGL_T_F32);
#pragma unroll
        for (int j = 0; j < 8; j++) n[j] += (double)p[j];
    }
}

// Sums over a wave through DPP and readlane (a shuffle would go through the LDS, twice for a double).
template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
    const int2 p = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(double, make_int2(dpp_i<CTRL>(p.x), dpp_i<CTRL>(p.y)));
}
__device__ __forceinline__ double rlane_d(double v, int l) {
    const int2 p = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_readlane(p.x, l), __builtin_amdgcn_readlane(p.y, l)));
}
__device__ __forceinline__ double row16_sum(double v) {
    v += dpp_d<0xB1>(v);
    v += dpp_d<0x4E>(v);
    v += dpp_d<0x141>(v);
    return v + dpp_d<0x140>(v);
}
// Sums over the threads of a row (a wave, or with WG the workgroup), in every one of them, in one order whatever the launch.
template <bool WG>
__device__ __forceinline__ double row_sum(double v, double *red) {
    v = row16_sum(v);
    v = (rlane_d(v, 0) + rlane_d(v, 16)) + (rlane_d(v, 32) + rlane_d(v, 48));
    if constexpr (WG) {
        __syncthreads();                       // the last round's reads are done
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        // lane l % 16 takes wave l % 16's sum (0 past the last wave)
        const int w = threadIdx.x & 15;
        v = rlane_d(row16_sum(w < (int)(blockDim.x >> 6) ? red[w] : 0.0), 0);
    }
    return v;
}
template <bool WG>
__device__ __forceinline__ uint32_t row_max(uint32_t v, double *red) {
    v = wave_max_u32(v);
    if constexpr (WG) {
        uint32_t *r = (uint32_t *)red;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
        __syncthreads();
        v = wave_max_u32(r[threadIdx.x & ((blockDim.x >> 6) - 1)]);
    }
    return v;
}

// mean and 1 / sqrt(... + eps) of a norm over the thread's values (0 past the row's end); rows: 1 / H
template <bool WG, typename Map>
__device__ __forceinline__ void norm_stats(int kind, const float (&v)[Map::N], const Map &m, float eps, double rows, double *red,
                                           double &mean, double &inv) {
    mean = 0.0;
    double q = 0.0;
    if (kind == BGL_NORM_LAYER) {
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < Map::N; k++) s += (double)v[k];
        mean = row_sum<WG>(s, red) * rows;
#pragma unroll
        for (int i = 0; i < Map::N / 8; i++) {
            const int n = m.has(i);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const double d = (double)v[8 * i + j] - mean;
                if (n >= 8 || j < n) q = fma(d, d, q);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < Map::N; k++) q = fma((double)v[k], (double)v[k], q);
    }
    inv = rsqrt(row_sum<WG>(q, red) * rows + (double)eps);
}

// NT 64: a wave a row, four in a workgroup of 256; 0: a workgroup a row, of as many threads as it has (one kernel for 256,
// 512 and 1024: as fast as one each, within a twentieth for rows normed twice).
template <int NT, int NV, int ROW>
__global__ __launch_bounds__(NT ? 256 : 1024) void k_norm(NormLaunch L) {
    constexpr bool WG = NT != 64;
    using Map = RowMap<NT, NV>;
    constexpr int N = Map::N;
    const bgl_norm &d = L.d;
    __shared__ double red[16];
    const int sub = WG ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Map m{WG ? (int)threadIdx.x : (int)(threadIdx.x & 63), d.H};
    const double rows = 1.0 / d.H;
    const long row = (long)blockIdx.x * (WG ? 1 : 4) + sub;
    if (row >= d.T) return;                                  // whole waves, which meet no barrier
    {
        float v[N], f[N];
#pragma unroll
        for (int i = 0; i < NV; i++) m.load(v + 8 * i, i, norm_row(d.x, row, d.ldx, d.x_type), d.x_type);
        if constexpr (ROW == ROW_GLU) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                m.load(f, i, norm_row(L.glu_u, row, d.ldx, BGL_T_F32), BGL_T_F32);
#pragma unroll
                for (int j = 0; j < 8; j++) v[8 * i + j] = i8_swiglu(v[8 * i + j], f[j]);      // of zeros: 0
            }
        }
        if constexpr (ROW == ROW_ADD || ROW == ROW_POST) {
#pragma unroll
            for (int i = 0; i < NV; i++) m.load(f + 8 * i, i, norm_row(d.f, row, d.ldf, d.f_type), d.f_type);
            double mean = 0.0, inv = 1.0;
            if constexpr (ROW == ROW_POST) norm_stats<WG>(d.post, f, m, d.post_eps, rows, red, mean, inv);
#pragma unroll
            for (int i = 0; i < NV; i++) {
                float *const vi = v + 8 * i;
                if (ROW == ROW_ADD && !d.gate) {             // one rounding without the way through double
#pragma unroll
                    for (int j = 0; j < 8; j++) vi[j] = fmaf(d.alpha, f[8 * i + j], vi[j]);
                } else {
                    double n[8];
                    if constexpr (ROW == ROW_POST) norm_chunk(n, m, i, f + 8 * i, d.post, mean, inv, d.post_w, d.w_add, d.post_b);
                    else {
#pragma unroll
                        for (int j = 0; j < 8; j++) n[j] = (double)f[8 * i + j];
                    }
                    if (d.gate) {
                        float g[8];
                        if (d.gate_c) m.load(g, i, norm_row(d.gate, row, d.gate_t, d.f_type), d.f_type);
                        else {
                            const float g1 = i8_ld(d.gate, d.f_type, (size_t)row * d.gate_t);
#pragma unroll
                            for (int j = 0; j < 8; j++) g[j] = g1;
                        }
#pragma unroll
                        for (int j = 0; j < 8; j++) n[j] *= (double)g[j];
                    }
#pragma unroll
                    for (int j = 0; j < 8; j++) vi[j] = (float)fma((double)d.alpha, n[j], (double)vi[j]);
                    m.cut(vi, i);                            // a post norm's bias
                }
            }
        }
        if (ROW != ROW_X || d.x_out) {
            void *const to = d.x_out ? const_cast<void *>(norm_row(d.x_out, row, d.ldo, d.x_type)) : nullptr;
#pragma unroll
            for (int i = 0; i < NV; i++) m.template store<true>(to, d.x_type, v + 8 * i, i);
        }
        if (!d.y && !d.yq) return;
        if (d.kind != BGL_NORM_NONE) {
            double mean, inv;
            norm_stats<WG>(d.kind, v, m, d.eps, rows, red, mean, inv);
#pragma unroll
            for (int i = 0; i < NV; i++) {
                double n[8];
                norm_chunk(n, m, i, v + 8 * i, d.kind, mean, inv, d.w, d.w_add, d.b);
#pragma unroll
                for (int j = 0; j < 8; j++) v[8 * i + j] = (float)n[j];
                m.cut(v + 8 * i, i);
            }
        }
        if (d.y) {
#pragma unroll
            for (int i = 0; i < NV; i++) m.template store<false>(const_cast<void *>(norm_row(d.y, row, d.ldy, d.y_type)), d.y_type, v + 8 * i, i);
        }
        if (d.yq) {
            uint32_t mb = I8_MX0;
#pragma unroll
            for (int k = 0; k < N; k++) mb = max(mb, __float_as_uint(v[k]) & 0x7fffffffu);
            const I8Scale s = i8_scale(row_max<WG>(mb, red));
            if (m.lt == 0) d.yscale[row] = s.sc;
            int8_t *q = d.yq + (size_t)row * d.ldq;
            const int H16 = (d.H + 15) & ~15;              // the bytes up to the row's next multiple of 16 are zeroed
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const float *t = v + 8 * i;
                if (m.at(i) < H16)
                    m.put(q, i, 1, make_uint2(i8_pack4(i8_code(t[0], s), i8_code(t[1], s), i8_code(t[2], s), i8_code(t[3], s)),
                                              i8_pack4(i8_code(t[4], s), i8_code(t[5], s), i8_code(t[6], s), i8_code(t[7], s))));
            }
        }
    }
}

// Rows wider than 16384 or narrower than 8: 1024 threads a row, one value at a time, the row read again for each pass.
// Only the thread that wrote a value of x_out reads it back.
__global__ __launch_bounds__(1024) void k_norm_wide(NormLaunch L) {
    const bgl_norm &d = L.d;
    __shared__ double red[16];
    const int tid = threadIdx.x;
    {
        const long row = blockIdx.x;
        double fmean = 0.0, finv = 1.0;
        if (d.f && d.post != BGL_NORM_NONE) {
            if (d.post == BGL_NORM_LAYER) {
                double s = 0.0;
                for (int h = tid; h < d.H; h += 1024) s += (double)i8_ld(d.f, d.f_type, (size_t)row * d.ldf + h);
                fmean = row_sum<true>(s, red) / d.H;
            }
            double q = 0.0;
            for (int h = tid; h < d.H; h += 1024) {
                const double t = (double)i8_ld(d.f, d.f_type, (size_t)row * d.ldf + h) - fmean;
                q = fma(t, t, q);
            }
            finv = 1.0 / sqrt(row_sum<true>(q, red) / d.H + (double)d.post_eps);
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
        if (!d.y && !d.yq) return;
        double mean = 0.0, inv = 1.0;
        if (d.kind == BGL_NORM_LAYER) {
            double s = 0.0;
            for (int h = tid; h < d.H; h += 1024) s += (double)value(h);
            mean = row_sum<true>(s, red) / d.H;
        }
        if (d.kind != BGL_NORM_NONE) {
            double q = 0.0;
            for (int h = tid; h < d.H; h += 1024) {
                const double t = (double)value(h) - mean;
                q = fma(t, t, q);
            }
            inv = 1.0 / sqrt(row_sum<true>(q, red) / d.H + (double)d.eps);
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
        if (!d.yq) return;
        const I8Scale s = i8_scale(row_max<true>(mb, red));
        if (tid == 0) d.yscale[row] = s.sc;
        int8_t *q = d.yq + (size_t)row * d.ldq;
        for (int h = tid; h < ((d.H + 15) & ~15); h += 1024) q[h] = (int8_t)(h < d.H ? i8_code(out(h), s) : 0);
    }
}

// ================================================================================== host side
template <int ROW>
static void norm_go(const NormLaunch &L, hipStream_t st) {
    auto go = [&](auto kernel, int threads, int rows) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)(((long)L.d.T + rows - 1) / rows)), dim3(threads), 0, st, L);
    };
    // (4096 bf16 rows of 4096 with 16 values a thread 31.2 us, with 8 33.1; 2048 normed-twice rows of 8192 36.8 and 42.7; few
    // rows wait for one row's passes: 1 of 4096 4.1 and 3.5, 300 5.9 and 5.6, 1024 9.0 and 9.4)
    const int H = L.d.H;
    if (H < 8) return go(k_norm_wide, 1024, 1);
    if constexpr (ROW != ROW_GLU)                            // (an MLP that narrow takes a workgroup a row)
        if (H <= 512) return go(k_norm<64, 1, ROW>, 256, 4);
    if (H <= 2048) go(k_norm<0, 1, ROW>, 256, 1);
    else if (H <= 4096 && L.d.T <= 512) go(k_norm<0, 1, ROW>, 512, 1);
    else if (H <= 4096) go(k_norm<0, 2, ROW>, 256, 1);
    else if (H <= 8192) go(k_norm<0, 2, ROW>, 512, 1);
    else if (H <= 16384) go(k_norm<0, 2, ROW>, 1024, 1);
    else go(k_norm_wide, 1024, 1);
}

// A launch has less than 2^32 threads, and up to 1024 take a row.
#define NORM_ROWS (1 << 21)
static int norm_launch(bgl_ctx *c, const NormLaunch &all) {
    const bgl_norm &a = all.d;
    int tok = prof_begin(c, all.glu_u || a.kind == BGL_NORM_NONE ? 0 : 2);
    for (long t = 0; t < a.T; t += NORM_ROWS) {
        NormLaunch L = all;
        bgl_norm &d = L.d;
        d.T = (int)std::min<long>(NORM_ROWS, a.T - t);
        auto at = [&](const void *p, long ld, int type) { return p ? const_cast<char *>((const char *)p) + t * ld * i8_elem(type) : nullptr; };
        d.x = at(a.x, a.ldx, a.x_type);
        d.f = at(a.f, a.ldf, a.f_type);
        d.gate = at(a.gate, a.gate_t, a.f_type);
        d.x_out = at(a.x_out, a.ldo, a.x_type);
        d.y = at(a.y, a.ldy, a.y_type);
        if (a.yq) { d.yq = a.yq + t * a.ldq; d.yscale = a.yscale + t; }
        if (all.glu_u) L.glu_u = all.glu_u + t * a.ldx;
        if (L.glu_u) norm_go<ROW_GLU>(L, c->stream);
        else if (!d.f) norm_go<ROW_X>(L, c->stream);
        else if (d.post == BGL_NORM_NONE) norm_go<ROW_ADD>(L, c->stream);
        else norm_go<ROW_POST>(L, c->stream);
    }
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
    return norm_launch(c, L);
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
    return norm_launch(c, L);
}
