// bgl_heads.hip -- queries, keys and values on their way from the q/k/v products to attention: a norm over each head,
// the rotation by the token's position, and the keys and values as 4-bit codes in the pages of a cache.
//
//   n = x | x / sqrt(mean(x^2) + eps) w | (x - mean) / sqrt(var + eps) w         over the D values of a head
//   y_i = n_i c_i - n_j s_i,  y_j = n_j c_i + n_i s_i                            for the pairs (i, j) that are rotated
//   groups of 32: m = fp16(min), s = fp16((max - m) (1/15)), c = rint((x - m) / s), value fp16(c s + m)
//
// Bound by memory where tokens are many: 4096 tokens of 40 heads of 128 in bf16, norms and rotation, 18.0 us, 4.8 TB/s.  4096 tokens'
// keys and values of 8 heads into the cache take 13.5 us, 22 MB: the vector units issue 8.4 of them (doubles, codes), waves wait half
// of their time.  Layer norms of 16-bit outputs, in double, 31 us where RMS norms take 17; fp32 outputs 34 us, 4.9 TB/s.  Few tokens are a launch
// and a chain of loads, position, its row of the table, the head: 8 tokens of 48 heads 4.8 us.
// A code changes by one where a value lies within rounding of a border between codes.  So y is computed in double and rounded
// once to fp32, and from there each step is one fp32 operation: the codes are the formula's.  (gfx950 issues double
// multiply-adds at the rate of single ones.)
#include <string.h>

#include <algorithm>

#include "../../include/beglin_qgemv.h"
#include "bgl_i8.h"
#include "bgl_kv.h"

#define HIPCHK(expr)                                                                             \
    do {                                                                                         \
        hipError_t e_ = (expr);                                                                  \
        if (e_ != hipSuccess) return bgl_fail(BGL_E_HIP, "%s: %s", #expr, hipGetErrorString(e_)); \
    } while (0)

struct HeadsLaunch {
    bgl_heads d;
    bgl_kv c;
    const int32_t *slots;        // of the d.T tokens of this launch; null: no cache
    int nq, nk, nv;              // heads to do of each
    float one_over_f;            // 1 / D
    double one_over;
};

// Sums over the GL lanes of a head, in every one of them.
template <int GL>
__device__ __forceinline__ float hd_sum(float v) {
    v += dpp_f<0xB1>(v);
    v += dpp_f<0x4E>(v);
    v += dpp_f<0x141>(v);
    if (GL > 8) v += dpp_f<0x140>(v);
    if (GL > 16) v += __shfl_xor(v, 16);
    if (GL > 32) v += __shfl_xor(v, 32);
    return v;
}
template <int GL>
__device__ __forceinline__ double hd_sum(double v) {
    v += dpp_d<0xB1>(v);
    v += dpp_d<0x4E>(v);
    v += dpp_d<0x141>(v);
    if (GL > 8) v += dpp_d<0x140>(v);
    if (GL > 16) v += __shfl_xor(v, 16);
    if (GL > 32) v += __shfl_xor(v, 32);
    return v;
}

// What a lane needs of the rotation for its 8 values d0 .. d0 + 7: their cosines and sines (the sines of half's first values with
// their sign), and for half where the other value of each pair lies.
struct HdTurn {
    float c[8], s[8];
    int other;                   // first of the 8 partners
    bool on;                     // the values are rotated
};
__device__ __forceinline__ HdTurn hd_turn(const bgl_heads &d, const float *rope, int d0) {
    HdTurn t;
    t.other = d0;
    t.on = d.rot_kind != BGL_ROT_NONE && d0 < d.rot;
#pragma unroll
    for (int j = 0; j < 8; j++) { t.c[j] = 1.0f; t.s[j] = 0.0f; }
    if (!t.on) return t;
    const int h = d.rot / 2;
    if (d.rot_kind == BGL_ROT_HALF) {
        t.other = d0 < h ? d0 + h : d0 - h;
        const int i = d0 < h ? d0 : t.other;
        kv_load8(t.c, rope, BGL_T_F32, i);
        kv_load8(t.s, rope, BGL_T_F32, h + i);
#pragma unroll
        for (int j = 0; j < 8; j++) t.s[j] = d0 < h ? -t.s[j] : t.s[j];
    } else {
        const kv_mf4 c = *(const kv_mf4 *)(rope + d0 / 2), s = *(const kv_mf4 *)(rope + h + d0 / 2);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            t.c[2 * j] = t.c[2 * j + 1] = c[j];
            t.s[2 * j] = -s[j];
            t.s[2 * j + 1] = s[j];
        }
    }
    return t;
}
// The norm's factors of a lane's values and of their partners, but for what is added to all of them (nothing where there are no weights).
struct HdWeights {
    float w[8], pw[8], add;
};
__device__ __forceinline__ HdWeights hd_weights(const bgl_heads &d, const float *w, const HdTurn &t, int d0) {
    HdWeights g;
#pragma unroll
    for (int j = 0; j < 8; j++) g.w[j] = g.pw[j] = 1.0f;
    g.add = 0.0f;
    if (d.norm == BGL_NORM_NONE || !w) return g;
    kv_load8(g.w, w, BGL_T_F32, d0);
    kv_load8(g.pw, w, BGL_T_F32, t.other);
    g.add = d.w_add;
    return g;
}

// A row of a head, of which a lane has the 8 values x (0 for a lane behind D) and, for half, their partners px (0 where nothing is rotated):
//     y = (x w c + x' w' s) / sqrt(..)        with w' and x' the partner's
// In fp32 what x and x' are multiplied by is the same for every head.
struct HdFast {
    float a[8], b[8];
    bool on;
    __device__ __forceinline__ HdFast(const bgl_heads &d, const HdWeights &g, const HdTurn &t) {
        const float add = g.add;
        on = t.on;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            a[j] = (g.w[j] + add) * t.c[j];
            b[j] = ((d.rot_kind == BGL_ROT_PAIRS ? g.w[j ^ 1] : g.pw[j]) + add) * t.s[j];
        }
    }
};
// A 16-bit output needs no double (16 additions and multiplications err by 2^-20 at most), unless a norm takes a difference from the mean
// or hides a row of tiny values behind no eps.
static __host__ __device__ __forceinline__ bool hd_fast(const bgl_heads &d) {
    return d.out_type != BGL_T_F32 && (d.norm == BGL_NORM_NONE || (d.norm == BGL_NORM_RMS && d.eps >= 1e-20f));
}
template <int GL>
__device__ __forceinline__ void hd_row_fast(float (&y)[8], const HeadsLaunch &L, float (&x)[8], float (&px)[8], const HdFast &f) {
    const bgl_heads &d = L.d;
    float inv = 1.0f;
    if (d.norm != BGL_NORM_NONE) {
        float q = 0.0f, eps = d.eps;
#pragma unroll
        for (int j = 0; j < 8; j++) q = fmaf(x[j], x[j], q);
        q = hd_sum<GL>(q);
        if (__any(!(q < 1e30f))) {                       // squares near fp32's end (or NaN): all of it 2^-80 as large, where eps counts no more
            const float down = q < 1e30f ? 1.0f : 0x1p-80f;
            eps = q < 1e30f ? eps : 0.0f;
            q = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) { x[j] *= down; px[j] *= down; q = fmaf(x[j], x[j], q); }
            q = hd_sum<GL>(q);
        }
        inv = __builtin_amdgcn_rsqf(fmaf(q, L.one_over_f, eps));
    }
    if (d.rot_kind == BGL_ROT_HALF) {
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = fmaf(x[j], f.a[j], px[j] * f.b[j]) * inv;
    } else if (d.rot_kind == BGL_ROT_PAIRS) {
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = fmaf(x[j], f.a[j], (f.on ? x[j ^ 1] : 0.0f) * f.b[j]) * inv;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = x[j] * f.a[j] * inv;
    }
}
// Keeps what is the same for every head in fp32 registers: as doubles, made once, it takes twice as many.
__device__ __forceinline__ void hd_opaque(float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j++) asm volatile("" : "+v"(v[j]));
}
template <int GL>
__device__ __forceinline__ void hd_row(float (&y)[8], const HeadsLaunch &L, const float (&x)[8], const float (&px)[8], HdWeights &g, HdTurn &t) {
    const bgl_heads &d = L.d;
    hd_opaque(g.w);
    hd_opaque(g.pw);
    hd_opaque(t.c);
    hd_opaque(t.s);
    double v[8], pv[8], inv = 1.0;
#pragma unroll
    for (int j = 0; j < 8; j++) { v[j] = x[j]; pv[j] = px[j]; }
    if (d.norm == BGL_NORM_LAYER) {
        double mean = 0.0;
#pragma unroll
        for (int j = 0; j < 8; j++) mean += v[j];
        mean = hd_sum<GL>(mean) * L.one_over;
        const bool in = (int)(threadIdx.x & (GL - 1)) * 8 < d.D;
#pragma unroll
        for (int j = 0; j < 8; j++) { v[j] = in ? v[j] - mean : 0.0; pv[j] -= mean; }
    }
    if (d.norm != BGL_NORM_NONE) {
        double q = 0.0;
#pragma unroll
        for (int j = 0; j < 8; j++) q = fma(v[j], v[j], q);
        inv = rsqrt(fma(hd_sum<GL>(q), L.one_over, (double)d.eps));
    }
    const double add = (double)g.add;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] *= add != 0.0 ? (double)g.w[j] + add : (double)g.w[j];
    if (d.rot_kind == BGL_ROT_NONE) {
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = (float)(v[j] * inv);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) pv[j] = d.rot_kind == BGL_ROT_PAIRS ? v[j ^ 1] : pv[j] * (add != 0.0 ? (double)g.pw[j] + add : (double)g.pw[j]);
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const double turned = fma(v[j], (double)t.c[j], pv[j] * (double)t.s[j]);
        y[j] = (float)((t.on ? turned : v[j]) * inv);
    }
}

// The codes, 0 .. 15, of a lane's 8 values, whose group is those of the lane's quad, and the group's step and floor (s | m << 16).
__device__ __forceinline__ uint32_t hd_codes(float (&c)[8], const float (&x)[8]) {
    float bad = 0.0f, t[8];                              // bad: NaN if a value has no end
#pragma unroll
    for (int j = 0; j < 8; j++) {
        bad = fmaf(x[j], 0.0f, bad);
        t[j] = __builtin_amdgcn_fmed3f(x[j], -32768.0f, 32768.0f);
    }
    float lo = fminf(fminf(fminf(t[0], t[1]), fminf(t[2], t[3])), fminf(fminf(t[4], t[5]), fminf(t[6], t[7])));
    float hi = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
    lo = fminf(lo, dpp_f<0xB1>(lo)); lo = fminf(lo, dpp_f<0x4E>(lo));
    hi = fmaxf(hi, dpp_f<0xB1>(hi)); hi = fmaxf(hi, dpp_f<0x4E>(hi));
    bad += dpp_f<0xB1>(bad); bad += dpp_f<0x4E>(bad);
    const _Float16 m = (_Float16)lo;
    const float fm = (float)m;
    const _Float16 s = (_Float16)fmaxf(0.0f, __fmul_rn(__fsub_rn(hi, fm), 1.0f / 15.0f));
    const float fs = (float)s;
    // 1 / s to nearest: s has 11 bits, so the remainder is exact, its correction errs by 2^-46 of 1 / s, and no quotient of such an s lies
    // within 2^-36 of the middle between two fp32 values
    float r = __builtin_amdgcn_rcpf(fs);
    r = fmaf(fmaf(-fs, r, 1.0f), r, r);
    r = fs > 0.0f && bad == 0.0f ? r : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) c[j] = rintf(__builtin_amdgcn_fmed3f(__fmul_rn(__fsub_rn(t[j], fm), r), 0.0f, 15.0f));
    if (!(bad == 0.0f)) return 0x7e000000u;              // NaN, step 0
    return (uint32_t)__builtin_bit_cast(uint16_t, s) | (uint32_t)__builtin_bit_cast(uint16_t, m) << 16;
}

__device__ __forceinline__ void hd_put_k(uint8_t *rec, int D, int tok, int li, const float (&x)[8]) {
    float c[8];
    const uint32_t sm = hd_codes(c, x);
    const int G = D / 32, b = li / G, j = li - b * G;
    // values 1, 3 lie 16 bits above 0, 2, and 4 .. 7 8 bits above 0 .. 3
    const float lo = fmaf(fmaf(fmaf(c[6], 16.0f, c[4]), 16.0f, c[2]), 16.0f, c[0]), hi = fmaf(fmaf(fmaf(c[7], 16.0f, c[5]), 16.0f, c[3]), 16.0f, c[1]);
    ((uint32_t *)rec)[(b * KV_TILE + tok) * G + j] = (uint32_t)lo | (uint32_t)hi << 16;
    if ((li & 3) == 0) ((uint32_t *)(rec + kv_k_steps(D)))[(li >> 2) * KV_TILE + tok] = sm;
}
__device__ __forceinline__ void hd_put_v(uint8_t *rec, int D, int tok, int li, const float (&x)[8]) {
    float c[8];
    const uint32_t sm = hd_codes(c, x);
    const int b = tok >> 2, r = tok & 3;
    uint8_t *p = rec + kv_v_codes(D) + (b * (D / 2) + 4 * li) * 4 + r;
#pragma unroll
    for (int j = 0; j < 4; j++) p[4 * j] = (uint8_t)(uint32_t)fmaf(c[2 * j + 1], 16.0f, c[2 * j]);
    if ((li & 3) == 0) {
        uint16_t *q = (uint16_t *)(rec + kv_v_steps(D)) + ((li >> 2) * 4 + b) * 8 + (r & 1) * 2 + (r >> 1);
        q[0] = (uint16_t)sm;
        q[4] = (uint16_t)(sm >> 16);
    }
}

// The token of workgroup x of a launch over n tokens, in whole rows of 128 where there are as many: 16 neighbours, which share the cache
// lines of a record, go to one XCD (workgroups go round the eight), whose L2 then puts their bytes together.
static __device__ __forceinline__ int hd_token(int x, int n) { return n < 128 ? x : (x & ~127) + ((x & 7) << 4) + (x >> 3 & 15); }

// A workgroup takes a token, each GL lanes (D / 8 of them at work) one head after the other: rows that go to q_out and k_out, and what goes into
// the cache.  FAST: rows of hd_row_fast are among them, for few tokens, which are one launch.  Of many the fast rows are k_heads_fast's: the
// others' doubles would leave them half as many waves (4096 tokens of 40 heads, bf16: 49 us together).
template <int GL, bool FAST>
__global__ __launch_bounds__(256, 2) void k_heads(HeadsLaunch L) {
    const bgl_heads &d = L.d;
    const int t = hd_token(blockIdx.x, d.T), li = threadIdx.x & (GL - 1), per = (int)blockDim.x / GL;
    if (t >= d.T) return;
    const bool in = 8 * li < d.D;
    const int d0 = in ? 8 * li : 0;
    const int pos = d.rot_kind != BGL_ROT_NONE ? d.pos[t] : 0;
    const int slot = L.slots ? L.slots[t] : -1;
    const bool kept = slot >= 0 && slot < (long)L.c.pages * L.c.page;
    const int tok = kept ? slot % L.c.page % KV_TILE : 0;
    const float *const rope = d.rope + (size_t)pos * d.rot;
    if (d.rot_kind != BGL_ROT_NONE && (uint32_t)pos >= (uint32_t)d.n_pos) return;
    const int step = (int)gridDim.y * per, first = (int)blockIdx.y * per + (int)threadIdx.x / GL;
    HdTurn turn = hd_turn(d, rope, d0);
    auto load = [&](float (&x)[8], float (&px)[8], const void *p, long at) {
        kv_load8(x, p, d.type, at + d0);
        if (d.rot_kind == BGL_ROT_HALF && turn.on) kv_load8(px, p, d.type, at + turn.other);
        else {
#pragma unroll
            for (int j = 0; j < 8; j++) px[j] = 0.0f;
        }
        if (!in) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = 0.0f;
        }
    };
    int i = first;
    if (i < L.nq) {
        HdWeights g = hd_weights(d, d.q_w, turn, d0);
        const HdFast f(d, g, turn);
        const bool fast = FAST && hd_fast(d);
        for (; i < L.nq; i += step) {
            float x[8], px[8], y[8];
            load(x, px, d.q, t * d.ldq + i * d.hdq);
            if (fast) hd_row_fast<GL>(y, L, x, px, f);
            else hd_row<GL>(y, L, x, px, g, turn);
            if (in) kv_store8(d.q_out, d.out_type, t * d.ldqo + i * d.hdqo + d0, y);
        }
    }
    if (i < L.nq + L.nk) {
        HdWeights g = hd_weights(d, d.k_w, turn, d0);
        const HdFast f(d, g, turn);
        const bool fast = FAST && d.k_out && hd_fast(d);
        for (; i < L.nq + L.nk; i += step) {
            const int h = i - L.nq;
            float x[8], px[8], y[8];
            if (!d.k_out && !kept) continue;
            load(x, px, d.k, t * d.ldk + h * d.hdk);
            if (fast) hd_row_fast<GL>(y, L, x, px, f);
            else hd_row<GL>(y, L, x, px, g, turn);
            if (!in) continue;
            if (d.k_out) kv_store8(d.k_out, d.out_type, t * d.ldko + h * d.hdko + d0, y);
            else hd_put_k(kv_at(L.c, slot, h), d.D, tok, li, y);
        }
    }
    if (!kept || !in) return;
    for (; i < L.nq + L.nk + L.nv; i += step) {
        const int h = i - L.nq - L.nk;
        float y[8];
        kv_load8(y, d.v, d.type, t * d.ldv + h * d.hdv + d0);
        hd_put_v(kv_at(L.c, slot, h), d.D, tok, li, y);
    }
}

// 8 values of a row and their partners, as they lie in memory.
template <bool F32>
struct HdRaw {
    kv_mu4 x[1 + F32], p[1 + F32];
    __device__ __forceinline__ void load(const char *row, int d0, int other) {
#pragma unroll
        for (int e = 0; e <= F32; e++) {
            x[e] = ((const kv_mu4 *)(row + (F32 ? 4 : 2) * d0))[e];
            p[e] = ((const kv_mu4 *)(row + (F32 ? 4 : 2) * other))[e];
        }
    }
    static __device__ __forceinline__ void values(float (&v)[8], const kv_mu4 (&u)[1 + F32], int type) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if constexpr (F32) v[j] = __uint_as_float(u[j >> 2][j & 3]);
            else if (type == BGL_T_F16) v[j] = (float)__builtin_bit_cast(_Float16, (uint16_t)(u[0][j / 2] >> (16 * (j & 1))));
            else v[j] = __uint_as_float(j & 1 ? u[0][j / 2] & 0xffff0000u : u[0][j / 2] << 16);
        }
    }
};
// The rows of hd_row_fast alone, each on its way while the one before it is worked on (4096 tokens of 40 heads: 18.1 us, 19.2 without).
template <int GL, bool F32>
__global__ __launch_bounds__(256, 4) void k_heads_fast(HeadsLaunch L) {
    const bgl_heads &d = L.d;
    const int t = hd_token(blockIdx.x, d.T), li = threadIdx.x & (GL - 1), per = (int)blockDim.x / GL;
    if (t >= d.T) return;
    const bool in = 8 * li < d.D;
    const int d0 = in ? 8 * li : 0, q_end = L.nq, total = L.nq + L.nk, step = (int)gridDim.y * per;
    const int pos = d.rot_kind != BGL_ROT_NONE ? d.pos[t] : 0;
    if (d.rot_kind != BGL_ROT_NONE && (uint32_t)pos >= (uint32_t)d.n_pos) return;
    HdTurn turn = hd_turn(d, d.rope + (size_t)pos * d.rot, d0);
    constexpr int ES = F32 ? 4 : 2;
    const char *const q0 = (const char *)d.q + t * d.ldq * ES, *const k0 = (const char *)d.k + t * d.ldk * ES;
    const long hdq = d.hdq * ES, hdk = d.hdk * ES;
    auto row = [=](int i) {                              // the last one past it
        const int x = min(i, total - 1);
        return x < q_end ? q0 + x * hdq : k0 + (x - q_end) * hdk;
    };
    HdRaw<F32> raw;
    int i = (int)blockIdx.y * per + (int)threadIdx.x / GL;
    raw.load(row(i), d0, turn.other);
    auto go = [&](int end, const float *w, void *out, long ld, long hd, int first) {
        if (i >= end) return;
        const HdWeights g = hd_weights(d, w, turn, d0);
        const HdFast f(d, g, turn);
        for (; i < end; i += step) {
            float x[8], px[8], y[8];
            HdRaw<F32>::values(x, raw.x, d.type);
            HdRaw<F32>::values(px, raw.p, d.type);
            raw.load(row(i + step), d0, turn.other);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[j] = in ? x[j] : 0.0f;
                px[j] = turn.on ? px[j] : 0.0f;
            }
            hd_row_fast<GL>(y, L, x, px, f);
            if (in) kv_store8(out, d.out_type, t * ld + (i - first) * hd + d0, y);
        }
    };
    go(q_end, d.q_w, d.q_out, d.ldqo, d.hdqo, 0);
    go(total, d.k_w, d.k_out, d.ldko, d.hdko, q_end);
}

struct KvReadLaunch {
    bgl_kv c;
    const int32_t *slots;
    int n, type;
    void *k, *v;
    long ldk, hdk, ldv, hdv;
};
__device__ __forceinline__ float kv_value(uint32_t c, uint32_t s, uint32_t m) {
    const _Float16 a = (_Float16)(float)c, b = __builtin_bit_cast(_Float16, (uint16_t)s), e = __builtin_bit_cast(_Float16, (uint16_t)m);
    return (float)__builtin_fmaf16(a, b, e);
}
template <int GL>
__global__ __launch_bounds__(256) void k_kv_read(KvReadLaunch L) {
    const int t = hd_token(blockIdx.x, L.n), li = threadIdx.x & (GL - 1), d0 = 8 * li, D = L.c.D, G = D / 32;
    if (t >= L.n) return;
    const int slot = L.slots[t];
    if (slot < 0 || slot >= (long)L.c.pages * L.c.page || d0 >= D) return;
    const int tok = slot % L.c.page % KV_TILE, per = (int)blockDim.x / GL, step = (int)gridDim.y * per;
    for (int i = (int)blockIdx.y * per + (int)threadIdx.x / GL; i < 2 * L.c.heads; i += step) {
        const int h = i % L.c.heads;
        const uint8_t *rec = kv_at(L.c, slot, h);
        float y[8];
        if (i < L.c.heads) {
            if (!L.k) continue;
            const int b = li / G, j = li - b * G;
            const uint32_t w = ((const uint32_t *)rec)[(b * KV_TILE + tok) * G + j];
            const uint32_t sm = ((const uint32_t *)(rec + kv_k_steps(D)))[(li >> 2) * KV_TILE + tok];
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = kv_value(w >> ((e & 1) * 16 + (e >> 2) * 8 + (e >> 1 & 1) * 4) & 15u, sm, sm >> 16);
            kv_store8(L.k, L.type, t * L.ldk + h * L.hdk + d0, y);
        } else {
            if (!L.v) continue;
            const int b = tok >> 2, r = tok & 3;
            typedef unsigned int u4 __attribute__((ext_vector_type(4)));               // of all four tokens
            const u4 w = *(const u4 *)(rec + kv_v_codes(D) + (b * (D / 2) + 4 * li) * 4), z = *(const u4 *)(rec + kv_v_steps(D) + ((li >> 2) * 4 + b) * 16);
            const uint32_t s = (r & 1 ? z[1] : z[0]) >> (16 * (r >> 1)), m = (r & 1 ? z[3] : z[2]) >> (16 * (r >> 1));
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = kv_value(w[e >> 1] >> (8 * r + 4 * (e & 1)) & 15u, s, m);
            kv_store8(L.v, L.type, t * L.ldv + h * L.hdv + d0, y);
        }
    }
}

// ================================================================================== host side
// A launch has less than 2^32 threads, 256 of them a token and up to 16 workgroups of few tokens.
#define HD_TOKENS (1 << 20)
#define HD_MANY (1 << 14)         // heads of queries that are a launch of their own beside the cache's rows

// Threads a workgroup.  A wave by itself takes a token's heads one after the other, so that the token's position and its row of the table are
// waited for less often (4096 tokens: keys and values 13.5 us, 17.8 in workgroups of 256; 40 heads 18.8 and 20.8); few tokens start faster in few
// workgroups (1 token 3.4 us, 3.8 in waves).
static int hd_block(int T) { return T < 8 ? 256 : 64; }
// Workgroups a token: as many as it takes to do every head at once, while the launch leaves units idle.
static unsigned hd_tokens(int T) { return T < 128 ? T : (T + 127) / 128 * 128; }
static unsigned hd_parts(int T, int items, int per) {
    const int all = (items + per - 1) / per;
    return (unsigned)std::max(1, std::min(all, 4096 / std::max(1, T)));
}
template <typename F>
static void hd_lanes(int D, F go) {
    if (D <= 64) go(std::integral_constant<int, 8>{});
    else if (D <= 128) go(std::integral_constant<int, 16>{});
    else if (D <= 256) go(std::integral_constant<int, 32>{});
    else go(std::integral_constant<int, 64>{});
}

static int heads_launch(bgl_ctx *c, const HeadsLaunch &all) {
    const bgl_heads &a = all.d;
    const int tok = prof_begin(c, 2);
    for (long t = 0; t < a.T; t += HD_TOKENS) {
        HeadsLaunch L = all;
        L.one_over_f = 1.0f / a.D;
        L.one_over = 1.0 / a.D;
        bgl_heads &d = L.d;
        d.T = (int)std::min<long>(HD_TOKENS, a.T - t);
        auto at = [&](const void *p, long ld, int type) { return p ? (char *)p + t * ld * (long)i8_elem(type) : nullptr; };
        d.q = at(a.q, a.ldq, a.type); d.k = at(a.k, a.ldk, a.type); d.v = at(a.v, a.ldv, a.type);
        d.q_out = at(a.q_out, a.ldqo, a.out_type); d.k_out = at(a.k_out, a.ldko, a.out_type);
        if (a.pos) d.pos = a.pos + t;
        if (all.slots) L.slots = all.slots + t;
        hd_lanes(d.D, [&](auto gl) {
            constexpr int GL = decltype(gl)::value;
            const int block = hd_block(d.T);
            auto go = [&](auto kernel, int nq, int nk, int nv) {
                L.nq = nq; L.nk = nk; L.nv = nv;
                hipLaunchKernelGGL(kernel, dim3(hd_tokens(d.T), hd_parts(d.T, nq + nk + nv, block / GL)), dim3((unsigned)block), 0, c->stream, L);
            };
            const bool q_fast = all.nq && hd_fast(d), k_fast = all.nk && d.k_out && hd_fast(d), exact = all.nv || (all.nq && !q_fast) || (all.nk && !k_fast);
            auto go_fast = [&](int nq, int nk) {
                if (d.type == BGL_T_F32) go(k_heads_fast<GL, true>, nq, nk, 0);
                else go(k_heads_fast<GL, false>, nq, nk, 0);
            };
            if (!exact) go_fast(all.nq, all.nk);
            else if (!q_fast) go(k_heads<GL, false>, all.nq, all.nk, all.nv);
            else if ((long)a.T * all.nq < HD_MANY) go(k_heads<GL, true>, all.nq, all.nk, all.nv);
            else {
                go_fast(all.nq, 0);
                go(k_heads<GL, false>, 0, all.nk, all.nv);
            }
        });
    }
    prof_end(c, tok);
    HIPCHK(hipGetLastError());
    return 0;
}

bool kv_rows_ok(long ld, long hd, long n, long heads, long D) {
    if (ld < 0 || hd < 0) return false;
    if (n == 1) return heads == 1 || hd >= D;
    if (heads == 1) return ld >= D;
    return (hd >= D && ld >= (heads - 1) * hd + D) || (ld >= D && hd >= (n - 1) * ld + D);
}
static bool type_ok(int t) { return t == BGL_T_F32 || t == BGL_T_F16 || t == BGL_T_BF16; }

int kv_check(const char *who, const bgl_kv *kv) {
    if (!kv || !kv->data) return bgl_fail(BGL_E_ARG, "%s: NULL cache", who);
    if (!bgl_kv_bytes(kv->pages, kv->page, kv->heads, kv->D))
        return bgl_fail(BGL_E_ARG, "%s: no cache of %d pages of %d tokens (a multiple of 16), %d heads of %d values (64, 96, 128, 192, 256)", who,
                        kv->pages, kv->page, kv->heads, kv->D);
    if ((uintptr_t)kv->data % 16) return bgl_fail(BGL_E_ARG, "%s: the cache is not 16-byte aligned", who);
    return 0;
}

extern "C" size_t bgl_kv_bytes(int pages, int page, int heads, int D) {
    if (pages < 1 || page < KV_TILE || page % KV_TILE || heads < 1 || heads > 65535 || !kv_dim_ok(D)) return 0;
    if ((long)pages * page > INT32_MAX) return 0;                  // slots are 32-bit
    return (size_t)pages * heads * (page / KV_TILE) * kv_record(D);
}

// What bgl_heads_dev and bgl_kv_append_dev ask of q, k and the rotation.
static int heads_check(const char *who, const bgl_heads *d) {
    if (d->T < 1 || d->D < 8 || d->D > 512 || d->D % 8) return bgl_fail(BGL_E_ARG, "%s: T=%d D=%d (a multiple of 8 up to 512)", who, d->T, d->D);
    if (!type_ok(d->type) || ((d->q_out || d->k_out) && !type_ok(d->out_type))) return bgl_fail(BGL_E_ARG, "%s: unknown element type", who);
    if (d->norm != BGL_NORM_NONE && d->norm != BGL_NORM_RMS && d->norm != BGL_NORM_LAYER) return bgl_fail(BGL_E_ARG, "%s: unknown norm kind", who);
    if (d->rot_kind != BGL_ROT_NONE && d->rot_kind != BGL_ROT_HALF && d->rot_kind != BGL_ROT_PAIRS)
        return bgl_fail(BGL_E_ARG, "%s: unknown rotation", who);
    if (d->rot_kind != BGL_ROT_NONE) {
        if (!d->rope || !d->pos || d->n_pos < 1) return bgl_fail(BGL_E_ARG, "%s: a rotation needs rope, pos and n_pos", who);
        if (d->rot < 8 || d->rot > d->D || d->rot % (d->rot_kind == BGL_ROT_HALF ? 16 : 8))
            return bgl_fail(BGL_E_ARG, "%s: rot=%d of %d values (a multiple of 16, or 8 for pairs)", who, d->rot, d->D);
    }
    if ((d->q != nullptr) != (d->q_out != nullptr)) return bgl_fail(BGL_E_ARG, "%s: q and q_out go together", who);
    if (d->q && (d->nq < 1 || d->nq > 65535)) return bgl_fail(BGL_E_ARG, "%s: nq=%d", who, d->nq);
    if (d->k && (d->nk < 1 || d->nk > 65535)) return bgl_fail(BGL_E_ARG, "%s: nk=%d", who, d->nk);
    if ((d->q && (!kv_rows_ok(d->ldq, d->hdq, d->T, d->nq, d->D) || !kv_rows_ok(d->ldqo, d->hdqo, d->T, d->nq, d->D))) ||
        (d->k && !kv_rows_ok(d->ldk, d->hdk, d->T, d->nk, d->D)) || (d->k_out && !kv_rows_ok(d->ldko, d->hdko, d->T, d->nk, d->D)) ||
        (d->v && !kv_rows_ok(d->ldv, d->hdv, d->T, d->nk, d->D)))
        return bgl_fail(BGL_E_ARG, "%s: rows of D=%d values overlap at these strides", who, d->D);
    if (d->q && d->q == d->q_out && (d->type != d->out_type || d->ldq != d->ldqo || d->hdq != d->hdqo))
        return bgl_fail(BGL_E_ARG, "%s: q_out is q with another type or stride", who);
    if (d->k_out && d->k == d->k_out && (d->type != d->out_type || d->ldk != d->ldko || d->hdk != d->hdko))
        return bgl_fail(BGL_E_ARG, "%s: k_out is k with another type or stride", who);
    if ((d->q_out && (d->q_out == d->k || d->q_out == d->v || d->q_out == d->k_out)) || (d->k_out && (d->k_out == d->q || d->k_out == d->v)))
        return bgl_fail(BGL_E_ARG, "%s: an output is one of the other rows", who);
    return 0;
}

extern "C" int bgl_heads_dev(bgl_ctx *c, const bgl_heads *d) {
    if (!c || !d) return bgl_fail(BGL_E_ARG, "bgl_heads_dev: NULL argument");
    if (!d->q && !d->k) return bgl_fail(BGL_E_ARG, "bgl_heads_dev: neither q nor k");
    if (d->v) return bgl_fail(BGL_E_ARG, "bgl_heads_dev: v is not used");
    if ((d->k != nullptr) != (d->k_out != nullptr)) return bgl_fail(BGL_E_ARG, "bgl_heads_dev: k and k_out go together");
    if (const int rc = heads_check("bgl_heads_dev", d)) return rc;
    HIPCHK(hipSetDevice(c->device));
    HeadsLaunch L;
    memset(&L, 0, sizeof L);
    L.d = *d;
    L.nq = d->q ? d->nq : 0;
    L.nk = d->k ? d->nk : 0;
    return heads_launch(c, L);
}

extern "C" int bgl_kv_append_dev(bgl_ctx *c, const bgl_kv *kv, const bgl_heads *d, const int32_t *slots) {
    if (!c || !d || !slots || !d->k || !d->v) return bgl_fail(BGL_E_ARG, "bgl_kv_append_dev: NULL argument");
    if (const int rc = kv_check("bgl_kv_append_dev", kv)) return rc;
    if (d->k_out) return bgl_fail(BGL_E_ARG, "bgl_kv_append_dev: k_out has to be NULL");
    if (const int rc = heads_check("bgl_kv_append_dev", d)) return rc;
    if (d->nk != kv->heads || d->D != kv->D)
        return bgl_fail(BGL_E_ARG, "bgl_kv_append_dev: %d heads of %d values into a cache of %d of %d", d->nk, d->D, kv->heads, kv->D);
    HIPCHK(hipSetDevice(c->device));
    HeadsLaunch L;
    memset(&L, 0, sizeof L);
    L.d = *d;
    L.c = *kv;
    L.slots = slots;
    L.nq = d->q ? d->nq : 0;
    L.nk = L.nv = d->nk;
    return heads_launch(c, L);
}

extern "C" int bgl_kv_read_dev(bgl_ctx *c, const bgl_kv *kv, const int32_t *slots, int n, void *k, long ldk, long hdk, void *v, long ldv,
                               long hdv, int type) {
    if (!c || !slots || (!k && !v)) return bgl_fail(BGL_E_ARG, "bgl_kv_read_dev: NULL argument");
    if (const int rc = kv_check("bgl_kv_read_dev", kv)) return rc;
    if (n < 1) return bgl_fail(BGL_E_ARG, "bgl_kv_read_dev: n=%d", n);
    if (!type_ok(type)) return bgl_fail(BGL_E_ARG, "bgl_kv_read_dev: unknown element type");
    if ((k && !kv_rows_ok(ldk, hdk, n, kv->heads, kv->D)) || (v && !kv_rows_ok(ldv, hdv, n, kv->heads, kv->D)) || k == v)
        return bgl_fail(BGL_E_ARG, "bgl_kv_read_dev: rows of D=%d values overlap", kv->D);
    HIPCHK(hipSetDevice(c->device));
    const int tok = prof_begin(c, 2);
    for (long t = 0; t < n; t += HD_TOKENS) {
        KvReadLaunch L;
        memset(&L, 0, sizeof L);
        L.c = *kv;
        L.slots = slots + t;
        L.n = (int)std::min<long>(HD_TOKENS, n - t);
        L.type = type;
        L.k = k ? (char *)k + t * ldk * (long)i8_elem(type) : nullptr; L.ldk = ldk; L.hdk = hdk;
        L.v = v ? (char *)v + t * ldv * (long)i8_elem(type) : nullptr; L.ldv = ldv; L.hdv = hdv;
        hd_lanes(kv->D, [&](auto gl) {
            constexpr int GL = decltype(gl)::value;
            hipLaunchKernelGGL((k_kv_read<GL>), dim3(hd_tokens(L.n), hd_parts(L.n, 2 * kv->heads, hd_block(L.n) / GL)), dim3((unsigned)hd_block(L.n)), 0, c->stream, L);
        });
    }
    prof_end(c, tok);
    HIPCHK(hipGetLastError());
    return 0;
}
