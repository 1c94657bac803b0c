// bgl_attn.h -- what the kernels of attention over the 4-bit cache share: the launch, which rows and keys belong
// together, the cache's codes as matrix-core operands, and the end of a row.
#pragma once
#include "bgl_kv.h"

typedef unsigned int at_u4 __attribute__((ext_vector_type(4)));

struct AttnLaunch {
    bgl_kv c;
    bgl_attn a;
    int g;                       // heads of q for one of the cache
    int ppt;                     // 16-token tiles a page
    uint32_t div_mul, div_shift; // t / ppt = (mulhi(t, div_mul) + t) >> div_shift for t < 2^31
    size_t page_bytes;           // of all heads
    int unit;                    // bgl_attn.hip: keys a unit, a multiple of AT_STEP
    int least;                   // bgl_attn.hip: units a workgroup, at least (1 or 2)
    int limit;                   // sequences with more than this many rows times g are another launch's
    float scale2;                // |scale| * log2(e); a negative scale turns q's sign
    float *part;                 // bgl_attn.hip's partial sums: [2 * workgroups] pieces
    int *sync;                   // for each workgroup that began a group of pieces, or an item: how many are written
};

// Weights are 2^8 exp2(s - m), where m is a row's largest score so far or up to 7 below it: m moves, and what was summed with it,
// only when a score passes it by more.  So weights stay below 2^15, and fp16 keeps 11 bits of all that are 2^-22 of the largest.
#define AT_P2 8.0f
#define AT_SLACK 7.0f

// A sequence: its rows (begin, n), its keys, and the range [lo, len) that one of its rows may see.
struct AttnSeq {
    int begin, n, len, lo;
};
__device__ __forceinline__ AttnSeq attn_seq(const AttnLaunch &L, int s) {
    AttnSeq q;
    const int b = L.a.start[s], e = L.a.start[s + 1], len = L.a.len[s];
    q.begin = min(max(b, 0), L.a.T);
    q.n = max(0, min(e, L.a.T) - q.begin);
    q.len = (int)min((long)max(len, 0), (long)L.a.ldt * L.c.page);
    q.lo = L.a.window ? (int)max(0l, (long)q.len - q.n - L.a.window + 1) : 0;
    q.lo = min(q.lo, q.len);
    return q;
}
// The keys [lo, hi] that token i of n sees (none: hi < lo).
__device__ __forceinline__ void attn_keys(const AttnLaunch &L, const AttnSeq &q, int i, int &lo, int &hi) {
    const int pos = q.len - q.n + i;
    hi = L.a.causal ? min(pos, q.len - 1) : q.len - 1;
    lo = L.a.window ? (int)max(0l, (long)pos - L.a.window + 1) : 0;
}

// ------------------------------------------------------------------ the cache's codes as operands
// fp16 pairs of the codes at bits 0 or 4 of each half of w (see bgl_kv.h), times s plus m, rounded once.  (The compiler takes two
// instructions for and + or with two constants, which cannot both be scalar operands.)
struct AtMagic {
    uint32_t lo, hi;                                     // in vector registers
    __device__ AtMagic() : lo(0x64006400u), hi(0x54005400u) { asm volatile("" : "+v"(lo), "+v"(hi)); }
};
__device__ __forceinline__ uint32_t at_and_or(uint32_t w, uint32_t mask, uint32_t with) {
    uint32_t r;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "s"(mask), "v"(with));
    return r;
}
__device__ __forceinline__ kv_h2 at_lo(const AtMagic &g, uint32_t w, kv_h2 s, kv_h2 m) {
    const kv_h2 c = __builtin_bit_cast(kv_h2, at_and_or(w, 0x000f000fu, g.lo)) - kv_h2{(_Float16)1024.0f, (_Float16)1024.0f};
    return __builtin_elementwise_fma(c, s, m);
}
__device__ __forceinline__ kv_h2 at_hi(const AtMagic &g, uint32_t w, kv_h2 s, kv_h2 m) {
    const kv_h2 c = __builtin_bit_cast(kv_h2, at_and_or(w, 0x00f000f0u, g.hi)) - kv_h2{(_Float16)64.0f, (_Float16)64.0f};
    return __builtin_elementwise_fma(c, s, m);
}
__device__ __forceinline__ kv_h8 at_join(kv_h2 a, kv_h2 b, kv_h2 c, kv_h2 d) {
    return kv_h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// 8 neighbouring values of a key from their dword and the group's (s, m)
__device__ __forceinline__ kv_h8 at_key(const AtMagic &g, uint32_t w, uint32_t sm) {
    const kv_h2 p = __builtin_bit_cast(kv_h2, sm), s = {p[0], p[0]}, m = {p[1], p[1]};
    return at_join(at_lo(g, w, s, m), at_hi(g, w, s, m), at_lo(g, w >> 8, s, m), at_hi(g, w >> 8, s, m));
}

__device__ __forceinline__ kv_f4 at_mfma(kv_h8 a, kv_h8 b, kv_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float at_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Maxima and sums over the four lanes of a wave that hold the same row (l, l ^ 16, l ^ 32, l ^ 48), in every one of them.
__device__ __forceinline__ float at_max4(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float at_sum4(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Dwords i .. of G at any 4-byte place.
template <int G>
__device__ __forceinline__ void at_dwords(uint32_t (&w)[G], const uint8_t *p) {
    typedef unsigned int u4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef unsigned int u2 __attribute__((ext_vector_type(2), aligned(4)));
#pragma unroll
    for (int i = 0; i + 4 <= G; i += 4) {
        const u4 v = *(const u4 *)(p + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; j++) w[i + j] = v[j];
    }
    constexpr int at = G / 4 * 4;
    if constexpr (G % 4 >= 2) {
        const u2 v = *(const u2 *)(p + 4 * at);
        w[at] = v[0];
        w[at + 1] = v[1];
    }
    if constexpr (G % 2) w[G - 1] = *(const uint32_t *)(p + 4 * (G - 1));
}

// Where token r of four stands in an operand of weights: 0, 2, 1, 3 is the order of V's pairs.
__device__ __forceinline__ constexpr int at_place(int r) { return (r & 1) * 2 + (r >> 1); }

// The smallest of a value over the 16 lanes of a row, as a scalar.
__device__ __forceinline__ int at_min16(int v) {
    v = min(v, dpp_i<0xB1>(v));
    v = min(v, dpp_i<0x4E>(v));
    v = min(v, dpp_i<0x141>(v));
    v = min(v, dpp_i<0x140>(v));
    return __builtin_amdgcn_readfirstlane(v);
}
// The same over the 32 lanes of either half.
__device__ __forceinline__ int pr_min32(int v) {
    v = min(v, dpp_i<0xB1>(v));
    v = min(v, dpp_i<0x4E>(v));
    v = min(v, dpp_i<0x141>(v));
    v = min(v, dpp_i<0x140>(v));
    return min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16));
}
// Sums of lanes 0 .. l.
__device__ __forceinline__ int at_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);                  // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);                  // lane 15 of rows 0 and 2 to rows 1 and 3
    return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);            // lane 31 to rows 2 and 3
}
// The page of the 16-token tile t of a sequence.
__device__ __forceinline__ int at_page(const AttnLaunch &L, int t) { return (int)(__umulhi((uint32_t)t, L.div_mul) + (uint32_t)t) >> L.div_shift; }

// A row of queries as operands: row r of the sequence's n * g (token r / g, head r % g of the group; past the last: the last), scaled by a power of
// two that puts the row's largest value in [2^14, 2^15): exact in fp16 down to 2^-28 of it (two parts for fp32 rows:
// 2^-22).  Values 8 G b .. + 8 G - 1 for a lane of block b of four (columns of 16), or with WIDE those of blocks b and 2 + b for a lane of half b
// (columns of 32).  PARTS is 2 for fp32 rows and 1 for the others.
template <int G, int PARTS, bool WIDE = false>
struct AtQuery {
    static constexpr int N = WIDE ? 2 : 1;
    kv_mu4 raw[N][G][PARTS];     // as they lie in memory: loaded early, waited for late

    __device__ __forceinline__ void load(const AttnLaunch &L, const AttnSeq &q, int head, int r, int b) {
        const int rr = min(r, q.n * L.g - 1), i = rr / L.g;
        const long at = (long)(q.begin + i) * L.a.ldq + (long)(head * L.g + rr - i * L.g) * L.a.hdq + 8 * G * b;
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int j = 0; j < G; j++) {
                const kv_mu4 *const p = (const kv_mu4 *)((const uint16_t *)L.a.q + PARTS * (at + 16 * G * n + 8 * j));
#pragma unroll
                for (int e = 0; e < PARTS; e++) raw[n][j][e] = p[e];
            }
    }
    __device__ __forceinline__ float value(int n, int j, int y, bool f16) const {
        if constexpr (PARTS == 2) return __uint_as_float(raw[n][j][y >> 2][y & 3]);
        const uint32_t w = raw[n][j][0][y >> 1] >> (16 * (y & 1)) & 0xffffu;
        return f16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)w) : __uint_as_float(w << 16);
    }
    // fac turns the products into scores of base 2, zero is where they begin (NaN for a row with a NaN or an infinity).
    __device__ __forceinline__ void operands(const AttnLaunch &L, kv_h8 (&qf)[N][PARTS][G], float &fac, float &zero) const {
        if (PARTS == 1 && L.a.type == BGL_T_F16) turn<true>(L, qf, fac, zero);
        else turn<false>(L, qf, fac, zero);
    }
    template <bool F16>
    __device__ __forceinline__ void turn(const AttnLaunch &L, kv_h8 (&qf)[N][PARTS][G], float &fac, float &zero) const {
        uint32_t top = 0;
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int j = 0; j < G; j++)
#pragma unroll
                for (int y = 0; y < 8; y++) top = max(top, __float_as_uint(value(n, j, y, F16)) & 0x7fffffffu);
        top = min(top, 0x7f800000u);                                                   // NaN counts as an infinity
        if constexpr (WIDE) {
            auto a = __builtin_amdgcn_permlane32_swap(top, top, false, false);
            top = max((uint32_t)a[0], (uint32_t)a[1]);
        } else {
            top = __float_as_uint(at_max4(__uint_as_float(top)));
        }
        const bool bad = top >= 0x7f800000u;
        const int e = bad ? 0 : min(14 - (max((int)(top >> 23), 1) - 127), 126);
        const float up = __int_as_float((127 + e) << 23) * (L.a.scale < 0.0f ? -1.0f : 1.0f);
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int j = 0; j < G; j++)
#pragma unroll
                for (int y = 0; y < 8; y++) {
                    const float v = value(n, j, y, F16) * up;
                    const _Float16 h = (_Float16)v;
                    qf[n][0][j][y] = h;
                    if constexpr (PARTS == 2) qf[n][1][j][y] = (_Float16)(v - (float)h);
                }
        // (a factor of 0 would make NaN of masked scores)
        fac = fmaxf(L.scale2 * __int_as_float((127 - e) << 23), 1e-30f);
        zero = bad ? NAN : 0.0f;
    }
};
// Keys e = 0, 1, .. behind a lane's first, of which a row sees those in [lo, hi]: the score, or -infinity.  (Integer operations on
// vector registers: comparisons would hold a scalar mask for each key.)
__device__ __forceinline__ int at_hides(int e, int lo, int hi) { return ((hi - e) | (e - lo)) >> 31; }
__device__ __forceinline__ float at_hide(float s, int hides) {
    return __uint_as_float((__float_as_uint(s) & ~(uint32_t)hides) | (0xff800000u & (uint32_t)hides));
}
// The same keys as a bit each, in the order of a weights' operand: those of two tiles that are seen.
__device__ __forceinline__ uint32_t at_seen(int lo, int hi, int tile) {
    uint32_t bits = 0;
#pragma unroll
    for (int x = 0; x < 8; x++) bits |= (uint32_t)(1 + at_hides(16 * (tile + (x >> 2)) + (x & 3), lo, hi)) << (4 * (x >> 2) + at_place(x & 3));
    return bits;
}
// [lo, hi] of a row, counted from a lane's first key; difference of any two ints held to where at_hides is right
__device__ __forceinline__ int at_from(int edge, int key) { return (int)min(max((long)edge - key, -(1l << 20)), 1l << 20); }
// fp16 ones where a bit of the eight is set
__device__ __forceinline__ kv_h8 at_ones(uint32_t bits) {
    kv_h8 v;
#pragma unroll
    for (int y = 0; y < 8; y++) v[y] = bits >> y & 1 ? (_Float16)1.0f : (_Float16)0.0f;
    return v;
}

// ------------------------------------------------------------------ NaN among the values
// A NaN times a weight of 0 is NaN: where rows of a product see different keys, V's NaN (a floor that is one) are multiplied as 0, and the
// rows that see them get theirs once the sums are done, in one more pass over the floors.
// Whether one of a lane's floors is NaN; it and its step's codes then count as 0.
__device__ __forceinline__ bool at_clean(at_u4 &z) {
    bool nan = false;
#pragma unroll
    for (int y = 2; y < 4; y++) {
        const uint32_t lo = (z[y] & 0x7c00u) == 0x7c00u ? 0xffffu : 0u, hi = (z[y] & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u;
        nan |= (lo | hi) != 0;
        z[y] &= ~(lo | hi);                              // (a NaN's step is 0)
    }
    return nan;
}
// Keys key .. key + 31: NaN into the sums of the rows that see one of V's.
template <int G, int NT>
__device__ __forceinline__ void at_nan(const AttnLaunch &L, const AttnSeq &q, int head, ucint table, int key, int lane, const int (&lo)[NT], const int (&hi)[NT],
                                       kv_f4 (&o)[NT][2 * G]) {
    const int col = lane & 15, b = lane >> 4;
    uint32_t bits[2] = {0, 0};                           // of the lane's first and last group
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int t = (key >> 4) + h, pg = 16 * t < q.len ? table[at_page(L, t)] : -1;
        if ((uint32_t)pg >= (uint32_t)L.c.pages) continue;
        const uint8_t *p = (const uint8_t *)L.c.data + (((size_t)pg * L.c.heads + head) * L.ppt + (t - at_page(L, t) * L.ppt)) * (20 * 32 * G);
        const at_u4 *vs = (const at_u4 *)(p + 18 * 32 * G);
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const at_u4 z = vs[((G * col + (x ? G - 1 : 0)) >> 4) * 4 + b];
#pragma unroll
            for (int y = 0; y < 4; y++)
                if ((z[2 + (y >> 1)] >> (16 * (y & 1)) & 0x7c00u) == 0x7c00u && 16 * t + 4 * b + at_place(y) < q.len) bits[x] |= 1u << (4 * h + y);
        }
    }
    if (!__any((bits[0] | bits[1]) != 0)) return;
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const kv_h8 seen = at_ones(at_seen(at_from(lo[t], key + 4 * b), at_from(hi[t], key + 4 * b), 0));
#pragma unroll
        for (int j = 0; j < G; j++) {
            const kv_f4 n = at_mfma(at_ones((G * col + j) >> 4 != G * col >> 4 ? bits[1] : bits[0]), seen, kv_f4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const float add = n[y] > 0.0f ? NAN : 0.0f;
                o[t][2 * j][y] += add;
                o[t][2 * j + 1][y] += add;
            }
        }
    }
}

// ------------------------------------------------------------------ a row's end
// What the sum of values (weights 2^8 exp2(s - M)) is multiplied by: 1 / (their sum + the sink's weight); 0 for a row without a key.
__device__ __forceinline__ float attn_factor(float M, float sum, bool sink, float sink2) {
    if (!sink) return M == -INFINITY && sum == 0.0f ? 0.0f : 1.0f / sum;
    const float top = fmaxf(M, sink2);
    if (top == -INFINITY && sum == 0.0f) return 0.0f;
    const float f = M == -INFINITY ? 0.0f : at_exp2(M - top);
    return f / (sum * f + (sink2 == INFINITY ? INFINITY : at_exp2(sink2 - top + AT_P2)));
}

// The prompt kernel (bgl_attn_p.hip): the call's sequences with more than L.limit rows times g, L.limit < INT32_MAX.
int run_attn_prompt(bgl_ctx *c, const AttnLaunch &L);
// Whether it takes all of a call's sequences, as far as the call's hints tell.
bool attn_prompt_alone(const AttnLaunch &L);
