// bgl_attn_p.hip -- attention of many rows a sequence (prompts, chunks of them) over the paged cache in 4 bits: the same sums as
// bgl_attn.hip's, bound by the matrix cores and by the exponentials, not by the cache's bytes.
//
// A workgroup takes RB rows of a head's group (tokens times heads of q) and goes over the keys that they see, 64 or 128 at a time.
// Its waves turn those keys' codes into fp16 operands once for all rows, in LDS: a record's order is the operands'
// order, so lane l writes 16 bytes at 16 l and reads 16 bytes at 16 l, without a transposition.  Two
// buffers: the next keys are converted, and the ones after those loaded, while the matrix cores work on the present ones; one barrier a stage.
// Each wave has 32 rows, as columns of S^T = K Q^T and O^T = V^T P^T; what a lane has of S^T is its part of P^T's operand.
//
// 4096 bf16 tokens of 32 heads of 128 over 8 of the cache: 151 us among other launches, 910 TFLOP/s of the rows' own products (a library's product of
// 8192^3 runs at 1180); 160 to 184 us by itself time after time, when the clock falls.  By counters the matrix units are busy 45% of that time and the vector units issue 50%: two waves a SIMD, which is what
// 240 registers leave, hardly overlap them, and every instruction of the loop counts, scalar ones too (the same loop with 50 scalar
// instructions more a stage: 181 us).  Tried and slower: the two waves of a SIMD in turns, half a stage apart (185 us); a stage's scores
// between the products of the one before it; 16 x 16 tiles (190 us where these took 175); three waves a SIMD for heads of 64 (118 for 113).
#include <string.h>

#include <algorithm>

#include "../../include/beglin_qgemv.h"
#include "bgl_i8.h"
#include "bgl_attn.h"

#define HIPCHK(expr)                                                                             \
    do {                                                                                         \
        hipError_t e_ = (expr);                                                                  \
        if (e_ != hipSuccess) return bgl_fail(BGL_E_HIP, "%s: %s", #expr, hipGetErrorString(e_)); \
    } while (0)

struct PromptLaunch {
    AttnLaunch A;
    int parts;                   // parts that a block's keys are split into; more than one: pieces in A.part, joined by k_attn_join
};
// A piece of an item (a block of RB rows and a head) and part: out's sums [RB][D], then the rows' m and their sums of weights.
template <int D, int RB>
__device__ __forceinline__ float *prompt_piece(const PromptLaunch &P, uint32_t item, int part) {
    return P.A.part + ((size_t)item * P.parts + part) * (RB * (D + 2));
}
// The blocks of all sequences lie in one line, a sequence's from the last, which sees the most keys, to the first: block x of the line, or
// false behind its end.  Every wave counts them by itself, lane by lane, each lane (S + 63) / 64 sequences.
struct PromptBlock {
    int s, block;
    AttnSeq q;
};
template <int RB>
__device__ __forceinline__ bool prompt_block(const AttnLaunch &L, uint32_t x, PromptBlock &b) {
    const int S = L.a.S, per = (S + 63) / 64, lane = threadIdx.x & 63;
    auto count = [&](const AttnSeq &q) { return (long)q.n * L.g > L.limit ? (q.n * L.g + RB - 1) / RB : 0; };
    AttnSeq mine_q;
    mine_q.begin = mine_q.n = mine_q.len = mine_q.lo = 0;
    int mine = 0;
    bool back = false;                                   // starts go back: the blocks could be more than 32 bits count
    for (int s = lane * per; s < min(S, (lane + 1) * per); s++) {
        mine_q = attn_seq(L, s);
        mine += count(mine_q);
        back |= min(L.a.start[s + 1], L.a.T) < mine_q.begin;
    }
    const int upto = at_scan(mine);
    if (__any(back) || x >= (uint32_t)__builtin_amdgcn_readlane(upto, 63)) return false;
    const int at_lane = __popcll(__ballot((uint32_t)upto <= x));
    int left = (int)x - __builtin_amdgcn_readlane(upto - mine, at_lane);               // blocks between the sequence's first and x
    b.s = at_lane * per;
    b.q.begin = __builtin_amdgcn_readlane(mine_q.begin, at_lane);
    b.q.n = __builtin_amdgcn_readlane(mine_q.n, at_lane);
    b.q.len = __builtin_amdgcn_readlane(mine_q.len, at_lane);
    b.q.lo = __builtin_amdgcn_readlane(mine_q.lo, at_lane);
    if (per > 1) {
        while (true) {
            b.q = attn_seq(L, b.s);
            b.q.begin = __builtin_amdgcn_readfirstlane(b.q.begin);
            b.q.n = __builtin_amdgcn_readfirstlane(b.q.n);
            b.q.len = __builtin_amdgcn_readfirstlane(b.q.len);
            const int n = count(b.q);
            if (left < n) break;
            left -= n;
            b.s++;
        }
    }
    b.block = count(b.q) - 1 - left;
    return true;
}

// v_mfma_f32_32x32x16_f16: lane l has 8 values of the sum for row or column l % 32, those of its half h = l / 32; results i = 0 .. 15 are
// rows 8 (i / 4) + 4 h + i % 4 of column l % 32.
typedef float pr_f16 __attribute__((ext_vector_type(16)));
__device__ __forceinline__ pr_f16 pr_mfma(kv_h8 a, kv_h8 b, pr_f16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ pr_f16 pr_all(float v) { return pr_f16{v, v, v, v, v, v, v, v, v, v, v, v, v, v, v, v}; }
// the larger value of a lane and the other lane of its row (l ^ 32)
__device__ __forceinline__ float pr_max2(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

// WAVES 8: two a SIMD, stages of 128 keys, two halves.  4: one, with all of its registers, for wide heads and two parts, stages of 64.
template <int G, int WAVES, int PARTS>
struct Prompt {
    static constexpr int D = 32 * G, RB = 32 * WAVES, HALVES = WAVES / 4, ST = 64 * HALVES;
    static constexpr int KN = G % 3 == 0 || G > 4 ? 2 : 1, VN = G % 3 == 0 ? 2 : 1;    // groups of 32 that a lane's values lie in, at most
    struct Shared {
        kv_h8 k[2][2 * HALVES][2 * G][64];               // [buffer][32 keys][of the sum over values, 16 at a time]
        kv_h8 v[2][4 * HALVES][G][64];                   // [buffer][16 keys, the sum][32 values]
        at_u4 flag[2][HALVES];                           // a tile each: 1 some value of V is NaN, 2 it has no page
    };
};

// at_nan (bgl_attn.h) for 32 rows: keys key .. key + 15.
template <int G>
__device__ __forceinline__ void pr_nan(const AttnLaunch &L, const AttnSeq &q, int head, ucint table, int key, int lane, int lo, int hi, pr_f16 (&o)[G]) {
    const int n = lane & 15, h = lane >> 5, t = key >> 4, pg = key < q.len ? table[at_page(L, t)] : -1;
    if ((uint32_t)pg >= (uint32_t)L.c.pages) return;
    const uint8_t *p = (const uint8_t *)L.c.data + (((size_t)pg * L.c.heads + head) * L.ppt + (t - at_page(L, t) * L.ppt)) * (20 * 32 * G);
    const at_u4 *vs = (const at_u4 *)(p + 18 * 32 * G);
    uint32_t bits[2] = {0, 0};                           // of the lane's first and last group
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const at_u4 z = vs[((G * n + (x ? G - 1 : 0)) >> 4) * 4 + 2 * u + h];
#pragma unroll
            for (int y = 0; y < 4; y++)
                if ((z[2 + (y >> 1)] >> (16 * (y & 1)) & 0x7c00u) == 0x7c00u && key + 8 * u + 4 * h + at_place(y) < q.len) bits[x] |= 1u << (4 * u + y);
        }
    if (!__any((bits[0] | bits[1]) != 0)) return;
    const int from = at_from(lo, key + 4 * h), to = at_from(hi, key + 4 * h);
    uint32_t seen = 0;
#pragma unroll
    for (int x = 0; x < 8; x++) seen |= (uint32_t)(1 + at_hides(8 * (x >> 2) + (x & 3), from, to)) << (4 * (x >> 2) + at_place(x & 3));
#pragma unroll
    for (int j = 0; j < G; j++) {
        const pr_f16 c = pr_mfma(at_ones((G * n + j) >> 4 != G * n >> 4 ? bits[1] : bits[0]), at_ones(seen), pr_all(0.0f));
#pragma unroll
        for (int i = 0; i < 16; i++) o[j][i] += c[i] > 0.0f ? NAN : 0.0f;
    }
}

template <int G, int WAVES, int PARTS>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 || (PARTS == 1 && G <= 4) ? 2 : 1) void k_attn_prompt(PromptLaunch P) {
    using T = Prompt<G, WAVES, PARTS>;
    constexpr int D = T::D, RB = T::RB, ST = T::ST, HALVES = T::HALVES, KN = T::KN, VN = T::VN;
    const AttnLaunch &L = P.A;
    __shared__ typename T::Shared sh;
    // Workgroup -> head (neighbouring workgroups, and with 8 heads a head an XCD, whose L2 holds its keys), part, block of the line.
    const uint32_t heads = (uint32_t)L.c.heads, rest = blockIdx.x / heads, line = rest / (uint32_t)P.parts;
    const int head = (int)(blockIdx.x - rest * heads), part = (int)(rest - line * (uint32_t)P.parts);
    PromptBlock at;
    if (!prompt_block<RB>(L, line, at)) return;
    const AttnSeq &q = at.q;
    const int rows = q.n * L.g, block = at.block;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, b = lane >> 4, h = lane >> 5;
    const AtMagic magic;
    // In the loop over keys the table is read by vector loads: a scalar load on its way makes every wait for the LDS a wait for all of it.
    const int *table = L.a.table + (size_t)at.s * L.a.ldt;
    int zero_lane = 0;
    asm volatile("" : "+v"(zero_lane));
    const int last_page = at_page(L, max(0, q.len - 1) >> 4);
    const int tile = wave;                               // of each stage's, whose K and V the wave converts
    const uint32_t kc_at = lane * (4 * G), vc_at = 10 * D + kc_at;
    auto ks_at = [&](int x) { return (uint32_t)(8 * D + (((G * b + x * (G - 1)) >> 2) * 16 + col) * 4); };       // of the first or last group
    auto vs_at = [&](int x) { return (uint32_t)(18 * D + (((G * col + x * (G - 1)) >> 4) * 4 + b) * 16); };
    // the keys of the block's rows, this part's stages among them
    int lo_first, lo_last, hi_first, hi_last;
    attn_keys(L, q, block * RB / L.g, lo_first, hi_first);
    attn_keys(L, q, (min(block * RB + RB, rows) - 1) / L.g, lo_last, hi_last);
    const int key0 = lo_first & ~15, stages = max(0, (hi_last + 1 - key0 + ST - 1) / ST);
    const int st0 = __builtin_amdgcn_readfirstlane((int)((long)stages * part / P.parts));
    const int st1 = __builtin_amdgcn_readfirstlane((int)((long)stages * (part + 1) / P.parts));

    auto key_of = [&](int stage) { return key0 + stage * ST + 16 * tile; };
    // the table's entry for the wave's tile of a stage, and where the tile lies in its page
    uint32_t in_page = 0;
    auto entry = [&](int stage) {
        const int t = key_of(stage) >> 4, p = at_page(L, t);
        in_page = (uint32_t)(t - p * L.ppt) * (20 * D);
        return table[min(p, last_page) + zero_lane];
    };
    auto page = [&](int stage, int e) {              // the page, or -1: past the keys, or none
        e = __builtin_amdgcn_readfirstlane(e);
        return key_of(stage) < q.len && (uint32_t)e < (uint32_t)L.c.pages ? e : -1;
    };
    uint32_t kc[G], ks[KN], vc[G];
    at_u4 vs[VN];
    const uint8_t *const records = (const uint8_t *)L.c.data + (size_t)head * L.ppt * (20 * D);
    // (a tile without a page loads one of the first page, and none of it counts)
    auto load_k = [&](int pg, uint32_t in) {
        const uint8_t *p = records + (size_t)(uint32_t)max(pg, 0) * L.page_bytes + in;
        at_dwords<G>(kc, p + kc_at);
#pragma unroll
        for (int x = 0; x < KN; x++) ks[x] = *(const uint32_t *)(p + ks_at(x));
    };
    auto load_v = [&](int pg, uint32_t in) {
        const uint8_t *p = records + (size_t)(uint32_t)max(pg, 0) * L.page_bytes + in;
        at_dwords<G>(vc, p + vc_at);
#pragma unroll
        for (int x = 0; x < VN; x++) vs[x] = *(const at_u4 *)(p + vs_at(x));
    };
    auto convert_k = [&](int buf) {
#pragma unroll
        for (int j = 0; j < G; j++)
            sh.k[buf][tile >> 1][(b >> 1) * G + j][(b & 1) * 32 + (tile & 1) * 16 + col] =
                at_key(magic, kc[j], KN == 2 && (G * b + j) >> 2 != G * b >> 2 ? ks[KN - 1] : ks[0]);
    };
    auto convert_v = [&](int buf, int stage, int pg) {
        uint32_t flag = pg < 0 ? 2 : 0;
        if (pg < 0 || key_of(stage) + 16 > q.len) {      // what lies behind the last key may be anything: 0
            asm volatile("");
            const int left = pg < 0 ? 0 : q.len - key_of(stage) - 4 * b;               // of the lane's four keys
            const uint32_t e = (left > 0 ? 0x0000ffffu : 0u) | (left > 2 ? 0xffff0000u : 0u);
            const uint32_t f = (left > 1 ? 0x0000ffffu : 0u) | (left > 3 ? 0xffff0000u : 0u);
#pragma unroll
            for (int x = 0; x < VN; x++) vs[x] &= at_u4{e, f, e, f};
        }
        // a floor whose exponent is all ones carries into its sign
        uint32_t ones = 0;
#pragma unroll
        for (int x = 0; x < VN; x++)
#pragma unroll
            for (int y = 2; y < 4; y++) ones |= (vs[x][y] & 0x7c007c00u) + 0x04000400u;
        if (__any((ones & 0x80008000u) != 0)) {
            asm volatile("");
            flag |= 1;
#pragma unroll
            for (int x = 0; x < VN; x++) (void)at_clean(vs[x]);
        }
#pragma unroll
        for (int j = 0; j < G; j++) {
            const at_u4 z = VN == 2 && (G * col + j) >> 4 != G * col >> 4 ? vs[VN - 1] : vs[0];
            const kv_h2 s0 = __builtin_bit_cast(kv_h2, (uint32_t)z[0]), s1 = __builtin_bit_cast(kv_h2, (uint32_t)z[1]);
            const kv_h2 m0 = __builtin_bit_cast(kv_h2, (uint32_t)z[2]), m1 = __builtin_bit_cast(kv_h2, (uint32_t)z[3]);
            const uint32_t c = vc[j], d = c >> 8;
            typedef uint32_t u2 __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int e = 0; e < 2; e++) {
                u2 w;
                w[0] = __builtin_bit_cast(uint32_t, e ? at_hi(magic, c, s0, m0) : at_lo(magic, c, s0, m0));
                w[1] = __builtin_bit_cast(uint32_t, e ? at_hi(magic, d, s1, m1) : at_lo(magic, d, s1, m1));
                ((u2 *)&sh.v[buf][tile][j][(b & 1) * 32 + 16 * e + col])[b >> 1] = w;
            }
        }
        if (lane == 0) ((uint32_t *)&sh.flag[buf])[tile] = flag;
    };

    int pg = page(st0, entry(st0));
    load_k(pg, in_page);
    load_v(pg, in_page);
    int next = entry(st0 + 1);
    // the wave's rows, one a lane (and l ^ 32)
    const int row0 = block * RB + wave * 32;
    kv_h8 qf[PARTS][2 * G];
    float fac, zero, m = -INFINITY;
    int lo, hi;
    {
        AtQuery<G, PARTS, true> query;
        query.load(L, q, head, row0 + (lane & 31), h);
        attn_keys(L, q, min(row0 + (lane & 31), rows - 1) / L.g, lo, hi);
        kv_h8 half[2][PARTS][G];                     // of the lane's values 8 G (2 x + h) ..
        query.operands(L, half, fac, zero);
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int p = 0; p < PARTS; p++)
#pragma unroll
                for (int j = 0; j < G; j++) qf[p][x * G + j] = half[x][p][j];
    }
    pr_f16 o[G];
    float l = 0.0f;                                  // of the lane's half of the keys
#pragma unroll
    for (int j = 0; j < G; j++) o[j] = pr_all(0.0f);
    const int lo_max = -pr_min32(-lo), lo_min = pr_min32(lo), hi_min = pr_min32(hi);
    const int hi_max = row0 < rows ? -pr_min32(-hi) : -1;      // (a wave without rows has nothing to do)

    bool nan = false;                                // V has had one
    // A stage's operands in runs of four, each read from the LDS while the run before it is multiplied: K of both 32 keys side by side
    // (two sums that do not wait for each other), then V.
    kv_h8 f[2][4];
    auto read = [&](int buf, int half, int run) {
#pragma unroll
        for (int x = 0; x < 4; x++) {
            if (run < G) f[run & 1][x] = sh.k[buf][2 * half + (x & 1)][2 * run + (x >> 1)][lane];
            else f[run & 1][x] = sh.v[buf][4 * half + (4 * (run - G) + x) / G][(4 * (run - G) + x) % G][lane];
        }
    };
    auto work = [&](int buf, int half, int key) {        // 64 keys
        const at_u4 fl = sh.flag[buf][half];
        pr_f16 s[2];
#pragma unroll
        for (int run = 0; run < G; run++) {
            read(buf, half, run + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int x = 0; x < 4; x++)
#pragma unroll
                for (int p = 0; p < PARTS; p++)
                    s[x & 1] = pr_mfma(f[run & 1][x], qf[p][2 * run + (x >> 1)], run + p + (x >> 1) ? s[x & 1] : pr_all(zero));
        }
        const uint32_t flags = (uint32_t)__builtin_amdgcn_readfirstlane((int)(fl[0] | fl[1] << 2 | fl[2] << 4 | fl[3] << 6));
        if ((flags & 0xaa) || key < lo_max || key + 63 > hi_min) {
            asm volatile("");
            // A lane's scores are of keys 8 (x / 4) + x % 4 behind its first: a bit for each that is seen, those of [lo, hi].
            auto below = [&](int edge) {                 // bits of the keys below
                const int e = (int)min(max((long)edge - (key + 4 * h), 0l), 64l), n = 4 * (e >> 3) + min(e & 7, 4);
                return n > 31 ? ~0u : (1u << n) - 1;
            };
            uint32_t seen = below(hi + 1) & ~below(lo);
#pragma unroll
            for (int t = 0; t < 4; t++)
                if (flags >> (2 * t) & 2) seen &= ~(0xffu << (8 * t));
#pragma unroll
            for (int x = 0; x < 32; x++) s[x >> 4][x & 15] = at_hide(s[x >> 4][x & 15], ~((int)(seen << (31 - x)) >> 31));
        }
        float top = s[0][0];
#pragma unroll
        for (int x = 1; x < 32; x++) top = fmaxf(top, s[x >> 4][x & 15]);
        top *= fac;
        if (__any(top > m + AT_SLACK)) {
            const float to = fmaxf(m, pr_max2(top)), g = to == -INFINITY ? 1.0f : at_exp2(m - to);
            m = to;
            l *= g;
#pragma unroll
            for (int j = 0; j < G; j++) o[j] *= g;
        }
        kv_h8 pf[4][PARTS];                              // (one part for 16-bit rows: bgl_attn.hip has both sides)
        const float off = AT_P2 - (m == -INFINITY ? 0.0f : m);
#pragma unroll
        for (int x = 0; x < 32; x++) {
            const int at = 4 * (x >> 2 & 1) + at_place(x & 3);
            const float p = at_exp2(fmaf(s[x >> 4][x & 15], fac, off));
            pf[x >> 3][0][at] = (_Float16)p;
            if constexpr (PARTS == 2) pf[x >> 3][1][at] = (_Float16)(p - (float)pf[x >> 3][0][at]);
        }
        // (the instruction's additions cut off what its largest term has no place for: short sums, which are added to nearest)
        const kv_h2 one = {(_Float16)1.0f, (_Float16)1.0f};
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
            for (int p = 0; p < PARTS; p++)
#pragma unroll
                for (int y = 0; y < 8; y += 2) sum[c & 1] = __builtin_amdgcn_fdot2(kv_h2{pf[c][p][y], pf[c][p][y + 1]}, one, sum[c & 1], false);
        l += sum[0] + sum[1];
#pragma unroll
        for (int run = G; run < 2 * G; run++) {
            if (run + 1 < 2 * G) read(buf, half, run + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int p = 0; p < PARTS; p++)
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int c = (4 * (run - G) + x) / G, j = (4 * (run - G) + x) % G;
                    o[j] = pr_mfma(f[run & 1][x], pf[c][p], o[j]);
                }
        }
        if (flags & 0x55) nan = true;
    };

    // (without a stage: of a tile past the keys, or one that nothing reads)
    convert_k(0);
    convert_v(0, st0, pg);
    pg = page(st0 + 1, next);
    uint32_t in = in_page;
    load_k(pg, in);
    if (HALVES == 1) load_v(pg, in);
    next = entry(st0 + 2);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    int buf = 0;
#pragma clang loop unroll(disable)
    for (int st = st0; st < st1; st++, buf ^= 1) {
        const int key = key0 + st * ST;
#pragma unroll
        for (int half = 0; half < HALVES; half++) {
            const bool mine = key + 64 * half <= hi_max && key + 64 * half + 63 >= lo_min;
            if (mine) read(buf, half, 0);
            __builtin_amdgcn_sched_barrier(0);
            // the next stage's K, then its V (each loaded half a stage before)
            if (half == 0) {
                convert_k(buf ^ 1);
                if (HALVES == 2) load_v(pg, in);
            }
            if (half == HALVES - 1) {
                convert_v(buf ^ 1, st + 1, pg);
                pg = page(st + 2, next);
                in = in_page;
                load_k(pg, in);
                if (HALVES == 1) load_v(pg, in);
                next = entry(st + 3);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (mine) work(buf, half, key + 64 * half);
        }
        // LDS writes are done; loads that are on their way end in registers, which their uses wait for
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    if (nan)
        for (int key = key0 + st0 * ST; key < key0 + st1 * ST; key += 16)
            pr_nan<G>(L, q, head, uni(L.a.table + (size_t)at.s * L.a.ldt), key, lane, lo, hi, o);
    const int r = row0 + (lane & 31);
    if (r >= rows) return;
    const int i = r / L.g, q_head = head * L.g + r - i * L.g;
    const float sum = l + __shfl_xor(l, 32);
    // unit n = 8 x + 4 h + y holds values 2 G n .. : value 2 j + e is result 8 e + 4 x + y of o[j]
    if (P.parts > 1) {
        float *const to = prompt_piece<D, RB>(P, line * heads + head, part);
        const int rr = r - block * RB;
        if (h == 0) { to[RB * D + rr] = m; to[RB * D + RB + rr] = sum; }
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int y = 0; y < 4; y++)
#pragma unroll
                for (int j = 0; j < G; j++) {
                    typedef float f2 __attribute__((ext_vector_type(2)));
                    *(f2 *)(to + rr * D + 2 * G * (8 * x + 4 * h + y) + 2 * j) = f2{o[j][4 * x + y], o[j][8 + 4 * x + y]};
                }
        return;
    }
    const float f1 = attn_factor(m, sum, L.a.sink != nullptr, L.a.sink ? L.a.sink[q_head] * 1.44269504088896340736f : 0.0f);
    const long to = (long)(q.begin + i) * L.a.ldo + (long)q_head * L.a.hdo;
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
        for (int y = 0; y < 4; y++) {
            const long d = to + 2 * G * (8 * x + 4 * h + y);
            if constexpr (G % 4 == 0) {
#pragma unroll
                for (int j = 0; j < G; j += 4) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = o[j + (e >> 1)][8 * (e & 1) + 4 * x + y] * f1;
                    kv_store8(L.a.out, L.a.type, d + 2 * j, v);
                }
            } else if constexpr (G % 2 == 0) {
#pragma unroll
                for (int j = 0; j < G; j += 2)
                    kv_store4(L.a.out, L.a.type, d + 2 * j, kv_f4{o[j][4 * x + y], o[j][8 + 4 * x + y], o[j + 1][4 * x + y], o[j + 1][8 + 4 * x + y]} * f1);
            } else {
#pragma unroll
                for (int j = 0; j < G; j++) {
                    i8_st(L.a.out, L.a.type, (size_t)(d + 2 * j), o[j][4 * x + y] * f1);
                    i8_st(L.a.out, L.a.type, (size_t)(d + 2 * j + 1), o[j][8 + 4 * x + y] * f1);
                }
            }
        }
}

// The parts of split blocks: 256 threads for 256 / (D / 4) rows of an item at a time.
template <int D, int RB>
__global__ __launch_bounds__(256) void k_attn_join(PromptLaunch P) {
    const AttnLaunch &L = P.A;
    const uint32_t x = blockIdx.x, line = x / (uint32_t)L.c.heads;
    const int head = (int)(x - line * (uint32_t)L.c.heads);
    PromptBlock at;
    if (!prompt_block<RB>(L, line, at)) return;
    const AttnSeq &q = at.q;
    const int block = at.block;
    const int r = (int)blockIdx.y * (256 / (D / 4)) + (int)threadIdx.x / (D / 4), d = (int)threadIdx.x % (D / 4) * 4;
    if (r >= RB || (int)threadIdx.x >= 256 / (D / 4) * (D / 4) || block * RB + r >= q.n * L.g) return;
    float M = -INFINITY, sum = 0.0f;
    for (int p = 0; p < P.parts; p++) M = fmaxf(M, prompt_piece<D, RB>(P, x, p)[RB * D + r]);
    kv_f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int p = 0; p < P.parts; p++) {
        const float *const from = prompt_piece<D, RB>(P, x, p);
        const float m = from[RB * D + r], f = m == -INFINITY ? 0.0f : at_exp2(m - M);
        v += *(const kv_f4 *)(from + r * D + d) * f;
        sum += from[RB * D + RB + r] * f;
    }
    const int i = (block * RB + r) / L.g, h = head * L.g + (block * RB + r) - i * L.g;
    v *= attn_factor(M, sum, L.a.sink != nullptr, L.a.sink ? L.a.sink[h] * 1.44269504088896340736f : 0.0f);
    kv_store4(L.a.out, L.a.type, (long)(q.begin + i) * L.a.ldo + (long)h * L.a.hdo + d, v);
}

// ================================================================================== host side
// A launch's blocks of RB rows times heads, and the parts of their keys.
struct PromptShape {
    long items;
    int parts;
};
static PromptShape prompt_shape(const AttnLaunch &L, int G, int RB) {
    PromptShape h;
    // as many blocks as the call's rows can make: every sequence of this kernel's may have one that is not full
    const long rows = (long)L.a.T * L.g, most = std::min<long>(L.a.S, rows / ((long)L.limit + 1));
    h.items = ((rows - most) / RB + most) * L.c.heads;
    // Where blocks leave CUs idle their keys are split: 64 keys of a workgroup take some 1 + G / 4 us, the second launch 3 us, and a part's sums go
    // out and in at 4 MB a us.  (512 rows of 32 heads of 128 over 4096 keys: 94 us in one part, 60 in four; over 512 keys 23 and 28 in two.)
    const double keys = L.a.window ? std::min((double)L.a.max_len, (double)L.a.window + RB) : L.a.max_len, stages = std::max(1.0, keys / 64);
    double best = 0;
    h.parts = 1;
    for (int p = 1; p <= 16 && p * h.items <= (p > 1 ? 256 : p * h.items); p++) {
        const double us = stages / p * (1 + G / 4.0) + (p > 1 ? 3 + (double)rows * L.c.heads * p * (32 * G) * 8 / 4e6 : 0);
        if (p == 1 || us < best) {
            best = us;
            h.parts = p;
        }
    }
    return h;
}
template <int G, int WAVES, int PARTS>
static int prompt_go(bgl_ctx *c, const AttnLaunch &L, const PromptShape &h) {
    constexpr int RB = Prompt<G, WAVES, PARTS>::RB, D = 32 * G;
    PromptLaunch P;
    memset(&P, 0, sizeof P);
    P.A = L;
    P.parts = h.parts;
    if (!h.items) return 0;
    if (P.parts > 1) {
        if (const int rc = dbuf_reserve(c, c->attn_part, (size_t)h.items * P.parts * RB * (D + 2) * 4, false)) return rc;
        P.A.part = (float *)c->attn_part.p;
    }
    hipLaunchKernelGGL((k_attn_prompt<G, WAVES, PARTS>), dim3((unsigned)(h.items * P.parts)), dim3(64 * WAVES), 0, c->stream, P);
    if (P.parts > 1) {
        constexpr int per = 256 / (D / 4);
        hipLaunchKernelGGL((k_attn_join<D, RB>), dim3((unsigned)h.items, (RB + per - 1) / per), dim3(256), 0, c->stream, P);
    }
    return 0;
}
template <int G>
static int prompt_pick(bgl_ctx *c, const AttnLaunch &L) {
    if constexpr (G <= 4) {
        const PromptShape h = prompt_shape(L, G, 256);
        if (L.a.type != BGL_T_F32) {
            // Blocks that are one round at most and not split: of half the size they fill more CUs, or two of them share one (32 heads of 128,
            // prompts of 128, 512, 1024 and 2048 tokens: 13.5, 22.7, 37.5 and 70 us in blocks of 256 rows, 10.8, 19.5, 32.7 and 66 of 128; of 4096
            // tokens 164 and 188: each block converts its keys).
            if (h.parts == 1 && h.items <= 256) return prompt_go<G, 4, 1>(c, L, {prompt_shape(L, G, 128).items, 1});
            return prompt_go<G, 8, 1>(c, L, h);
        }
        if constexpr (G <= 3) return prompt_go<G, 8, 2>(c, L, h);
    }
    if constexpr (G > 3) {
        const PromptShape h = prompt_shape(L, G, 128);
        if constexpr (G > 4) {
            if (L.a.type != BGL_T_F32) return prompt_go<G, 4, 1>(c, L, h);
        }
        return prompt_go<G, 4, 2>(c, L, h);
    }
}

// What the prompt kernel costs, in us, for the sequences of more than `limit` rows times g if their rows see `keys` keys: rounds of blocks on the CUs,
// 64 keys at a time (0.7 (1 + G / 4) us measured with two waves a SIMD, half as much again with one) behind some 8 us, 6 more with a second launch.  From
// the hints, of the rows beside the longest sequence's as many for each of the others.
static double prompt_us(AttnLaunch L, int limit, double keys) {
    const int G = L.c.D / 32;
    const bool f32 = L.a.type == BGL_T_F32, wide = G > 4 || (G > 3 && f32);            // one wave a SIMD
    L.limit = limit;
    int RB = wide ? 128 : 256, cap = 256;
    const PromptShape h = prompt_shape(L, G, RB);
    if (!wide && !f32 && h.parts == 1 && h.items <= 256) { RB = 128; cap = 512; }      // (prompt_pick)
    const long most = std::min(L.a.T, std::max(1, L.a.max_rows)), others = (L.a.T - most) * L.g, S = L.a.S - 1, count = others > S * limit ? S : 0;
    const long items = ((most * L.g + RB - 1) / RB + (count ? count + std::max(0l, others - count) / RB : 0)) * L.c.heads * h.parts;
    if (L.a.window) keys = std::min(keys, (double)L.a.window + RB);
    return 8 + (items + cap - 1) / cap * std::max(1.0, keys / 64) / h.parts * (1 + G / 4.0) * (wide ? 1.05 : 0.7) + (h.parts > 1 ? 6 : 0);
}
// One launch for all sequences, or k_attn for those of few rows (some 15 us with its launch, and the keys at 5 MB a us)?  Their keys are as many as the
// longest sequence's for all that is known, but a prompt's may be its own rows only: the two costs' geometric mean stands for what two
// launches take, and a tenth more, so that either choice is wrong by little.  Of 165 calls, heads of 64 to 256, 2 to 32 sequences, the slower form is
// taken in 16 by more than 15%, at most by 54%; the rule before, S * heads <= 256 and 2048 keys at most: in 40, by up to 110%.  (32 heads over 8, us in one
// launch and in two.  bf16, heads of 128: 200 rows and 15 of one, 1000 keys each, 29 and 45; 300 rows of three, 300 keys, and 5 of one, 1500 keys, 43 and 28;
// 2000 rows and 31 of one, 3000 keys each, 147 and 130.  Heads of 256: 40 rows and 31 of one, 2048 keys each, 179 and 85.  fp32, heads of 128: the same 154 and 78.)
bool attn_prompt_alone(const AttnLaunch &L) {
    if (L.a.S == 1) return true;
    const long few = L.a.window ? std::min((long)L.a.max_len, L.a.window + 32l) : L.a.max_len;
    const double rest = 15 + (double)(L.a.S - 1) * few * L.c.heads * L.c.D * 1.25 / 5e6;
    const double one = prompt_us(L, 0, L.a.max_len), far = prompt_us(L, 32, L.a.max_len), near = prompt_us(L, 32, std::min(L.a.max_len, L.a.max_rows));
    return one * one <= 1.2 * (far + rest) * (near + rest);
}

int run_attn_prompt(bgl_ctx *c, const AttnLaunch &L) {
    switch (L.c.D / 32) {
    case 2: return prompt_pick<2>(c, L);
    case 3: return prompt_pick<3>(c, L);
    case 4: return prompt_pick<4>(c, L);
    case 6: return prompt_pick<6>(c, L);
    default: return prompt_pick<8>(c, L);
    }
}
