// bgl_attn_p.hip -- attention of many rows a sequence (prompts, chunks of them) over the paged cache in 4 bits: the same sums as
// bgl_attn.hip's, bound by the matrix cores and by the exponentials, not by the cache's bytes.
//
// A workgroup takes RB rows of a head's group (tokens times heads of q) and goes over the keys that they see, 64 at a time.
// Its waves turn those keys' codes into fp16 operands once for all rows, in LDS: a record's order is the operands'
// order, so lane l writes 16 bytes at 16 l and reads 16 bytes at 16 l, without a conflict and without a transposition.  Two
// buffers: the next 64 keys are converted, and the ones after those loaded, while the matrix cores work on the present ones.
// Each wave has 16 NT rows, as columns of S^T = K Q^T and O^T = V^T P^T; what a lane has of S^T is its part of P^T's operand.
// A row's sum of weights is one more product, with ones in V's place: the vector units are the narrower side here.
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
    int blocks;                  // row blocks a sequence and head in the grid; a workgroup takes every blocks-th from its first
    int parts;                   // parts that a block's keys are split into; more than one: pieces in A.part, joined by k_attn_join
};
// A piece of an item (block, sequence, head) and part: out's sums [RB][D], then the rows' m and their sums of weights.
template <int D, int RB>
__device__ __forceinline__ float *prompt_piece(const PromptLaunch &P, long item, int part) {
    return P.A.part + (item * P.parts + part) * (long)(RB * (D + 2));
}
// Workgroup -> head (neighbouring workgroups, and with 8 heads a head an XCD, whose L2 holds its keys), part, sequence, and block from the last,
// which sees the most keys, to the first.
struct PromptItem {
    int head, part, s, block;
    long item;
    __device__ PromptItem(const PromptLaunch &P, long x) {
        head = (int)(x % P.A.c.heads); x /= P.A.c.heads;
        part = (int)(x % P.parts); x /= P.parts;
        s = (int)(x % P.A.a.S); x /= P.A.a.S;
        block = P.blocks - 1 - (int)x;
        item = ((long)block * P.A.a.S + s) * P.A.c.heads + head;
    }
};

template <int G, int WAVES, int NT, int PARTS>
struct Prompt {
    static constexpr int D = 32 * G, RB = 16 * NT * WAVES, THREADS = 64 * WAVES, ST = 64;
    static constexpr bool K2 = G % 3 == 0 || G > 4, V2 = G % 3 == 0;                  // as in AttnRaw
    struct Shared {
        kv_h8 k[2][4][G][64], v[2][2][2 * G][64];
        uint32_t flag[2][4];                             // a tile: 1 some value of V is NaN, 2 it has no page
        uint32_t nan[2][4][G];                           // which of the 16 keys, for each group
    };
};

template <int G, int WAVES, int NT, int PARTS>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 ? 2 : 1) void k_attn_prompt(PromptLaunch P) {
    using T = Prompt<G, WAVES, NT, PARTS>;
    constexpr int D = T::D, RB = T::RB, ST = T::ST;
    constexpr bool K2 = T::K2, V2 = T::V2;
    const AttnLaunch &L = P.A;
    __shared__ typename T::Shared sh;
    const PromptItem it(P, blockIdx.x);
    AttnSeq q = attn_seq(L, it.s);
    q.begin = __builtin_amdgcn_readfirstlane(q.begin);
    q.n = __builtin_amdgcn_readfirstlane(q.n);
    q.len = __builtin_amdgcn_readfirstlane(q.len);
    const int rows = q.n * L.g;
    if ((long)q.n * L.g <= L.limit) return;              // another kernel's
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, b = lane >> 4;
    const ucint table = uni(L.a.table + (size_t)it.s * L.a.ldt);
    const AtMagic magic;
    auto none = [&](int pg) { return (uint32_t)pg >= (uint32_t)L.c.pages; };
    auto entry = [&](int key) { return key < q.len ? table[at_page(L, key >> 4)] : -1; };
    for (int block = it.block; block * RB < rows; block += P.blocks) {
        // the keys of the block's rows, this part's stages of 64 among them
        int lo_first, lo_last, hi_first, hi_last;
        attn_keys(L, q, block * RB / L.g, lo_first, hi_first);
        attn_keys(L, q, min(block * RB + RB, rows) / L.g - (min(block * RB + RB, rows) % L.g == 0), lo_last, hi_last);
        const int key0 = lo_first & ~15, stages = max(0, (hi_last + 1 - key0 + ST - 1) / ST);
        const int parts = block < P.blocks ? P.parts : 1;          // blocks that max_rows did not tell of have no room for pieces
        if (it.part >= parts) break;
        int st = __builtin_amdgcn_readfirstlane((int)((long)stages * it.part / parts));
        const int st1 = __builtin_amdgcn_readfirstlane((int)((long)stages * (it.part + 1) / parts));

        // A wave's share of a stage's conversion: one of the four tiles, both of it (4 waves) or K or V of it (8).
        const int tile = WAVES == 8 ? wave >> 1 : wave;
        const bool do_k = WAVES == 4 || !(wave & 1), do_v = WAVES == 4 || (wave & 1);
        uint32_t kc[G], ks[K2 ? 2 : 1], vc[G];
        at_u4 vs[V2 ? 2 : 1];
        auto key_of = [&](int stage) { return key0 + stage * ST + 16 * tile; };
        auto load = [&](int key, int pg) {
            const int t = key >> 4;
            const size_t rec = none(pg) ? 0 : ((size_t)pg * L.c.heads + it.head) * L.ppt + (t - at_page(L, t) * L.ppt);
            const uint8_t *p = (const uint8_t *)L.c.data + rec * (20 * D);
            if (do_k) {
                at_dwords<G>(kc, p + lane * (4 * G));
                const uint32_t *s = (const uint32_t *)(p + 8 * D);
                ks[0] = s[(G * b >> 2) * 16 + col];
                if constexpr (K2) ks[1] = s[((G * b + G - 1) >> 2) * 16 + col];
            }
            if (do_v) {
                at_dwords<G>(vc, p + 10 * D + lane * (4 * G));
                const at_u4 *s = (const at_u4 *)(p + 18 * D);
                vs[0] = s[(G * col >> 4) * 4 + b];
                if constexpr (V2) vs[1] = s[((G * col + G - 1) >> 4) * 4 + b];
            }
        };
        auto convert = [&](int buf, int key, int pg) {
            if (do_k) {
#pragma unroll
                for (int j = 0; j < G; j++) sh.k[buf][tile][j][lane] = at_key(magic, kc[j], K2 && (G * b + j) >> 2 != G * b >> 2 ? ks[K2] : ks[0]);
            }
            if (do_v) {
                uint32_t flag = none(pg) ? 2 : 0;
                const int left = none(pg) ? 0 : q.len - key - 4 * b;                   // of the lane's four keys
                if (none(pg) || key + 16 > q.len) {      // what lies behind the last key may be anything: 0
                    asm volatile("");
                    const uint32_t e = (left > 0 ? 0x0000ffffu : 0u) | (left > 2 ? 0xffff0000u : 0u);
                    const uint32_t f = (left > 1 ? 0x0000ffffu : 0u) | (left > 3 ? 0xffff0000u : 0u);
#pragma unroll
                    for (int x = 0; x < (V2 ? 2 : 1); x++) vs[x] &= at_u4{e, f, e, f};
                }
                bool nan = false;
#pragma unroll
                for (int x = 0; x < (V2 ? 2 : 1); x++)
#pragma unroll
                    for (int y = 2; y < 4; y++) nan |= (vs[x][y] & 0x7c00u) == 0x7c00u || (vs[x][y] & 0x7c000000u) == 0x7c000000u;
                if (__any(nan)) {                        // they reach the rows that see them, in the products' end
                    asm volatile("");
                    flag |= 1;
                    uint32_t bits[V2 ? 2 : 1];
#pragma unroll
                    for (int x = 0; x < (V2 ? 2 : 1); x++) {
                        bits[x] = 0;
#pragma unroll
                        for (int y = 0; y < 4; y++)
                            if ((vs[x][2 + (y >> 1)] >> (16 * (y & 1)) & 0x7c00u) == 0x7c00u) {
                                bits[x] |= 1u << y;
                                vs[x][2 + (y >> 1)] &= y & 1 ? 0x0000ffffu : 0xffff0000u;
                            }
                    }
                    // bit 4 b + y of group g; every lane of (b, g) says the same
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        uint32_t mine = (G * col >> 4) == g ? bits[0] << (4 * b) : 0u;
                        if constexpr (V2) mine |= ((G * col + G - 1) >> 4) == g ? bits[1] << (4 * b) : 0u;
#pragma unroll
                        for (int x = 1; x < 64; x <<= 1) mine |= (uint32_t)__shfl_xor((int)mine, x);
                        if (lane == 0) sh.nan[buf][tile][g] = mine;
                    }
                }
#pragma unroll
                for (int j = 0; j < G; j++) {
                    const at_u4 z = V2 && (G * col + j) >> 4 != G * col >> 4 ? vs[V2] : vs[0];
                    const kv_h2 s0 = __builtin_bit_cast(kv_h2, (uint32_t)z[0]), s1 = __builtin_bit_cast(kv_h2, (uint32_t)z[1]);
                    const kv_h2 m0 = __builtin_bit_cast(kv_h2, (uint32_t)z[2]), m1 = __builtin_bit_cast(kv_h2, (uint32_t)z[3]);
                    const uint32_t c = vc[j], d = c >> 8;
                    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        u2 w;
                        w[0] = __builtin_bit_cast(uint32_t, e ? at_hi(magic, c, s0, m0) : at_lo(magic, c, s0, m0));
                        w[1] = __builtin_bit_cast(uint32_t, e ? at_hi(magic, d, s1, m1) : at_lo(magic, d, s1, m1));
                        ((u2 *)&sh.v[buf][tile >> 1][2 * j + e][lane])[tile & 1] = w;
                    }
                }
                if (lane == 0) sh.flag[buf][tile] = flag;
            }
        };

        int pg = entry(key_of(st)), pn = entry(key_of(st + 1));
        if (st < st1) load(key_of(st), pg);
        // the wave's rows
        kv_h8 qf[NT][PARTS][G];
        float fac[NT], zero[NT], m[NT];
        int lo[NT], hi[NT], lo_max = 0, lo_min = INT32_MAX, hi_min = INT32_MAX, hi_max = -1;
        kv_f4 o[NT][2 * G], l[NT];
        const int row0 = block * RB + wave * 16 * NT;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            at_query<G, PARTS>(L, q, it.head, row0 + 16 * t + col, b, qf[t], fac[t], zero[t], lo[t], hi[t]);
            lo_max = max(lo_max, lo[t]);
            lo_min = min(lo_min, lo[t]);
            hi_min = min(hi_min, hi[t]);
            hi_max = max(hi_max, hi[t]);
            m[t] = -INFINITY;
            l[t] = kv_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < 2 * G; j++) o[t][j] = kv_f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        lo_max = -at_min16(-lo_max);
        lo_min = at_min16(lo_min);
        hi_min = at_min16(hi_min);
        hi_max = row0 < rows ? -at_min16(-hi_max) : -1;  // (a wave without rows has nothing to do)
        const kv_h8 ones = at_ones(0xff);

        auto work = [&](int buf, int blk, int key) {     // keys key .. key + 31
            const uint32_t f0 = sh.flag[buf][2 * blk], f1 = sh.flag[buf][2 * blk + 1];
            const uint32_t flags = (uint32_t)__builtin_amdgcn_readfirstlane((int)(f0 | f1 << 2));
            kv_f4 s[NT][2];
#pragma unroll
            for (int t = 0; t < NT; t++) s[t][0] = s[t][1] = kv_f4{zero[t], zero[t], zero[t], zero[t]};
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int j = 0; j < G; j++) {
                    const kv_h8 k = sh.k[buf][2 * blk + h][j][lane];
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int p = 0; p < PARTS; p++) s[t][h] = at_mfma(k, qf[t][p][j], s[t][h]);
                }
            uint32_t hidden[NT];
            if ((flags & 10) || key < lo_max || key + 31 > hi_min) {
                asm volatile("");
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    hidden[t] = 0;
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const int k = key + 16 * h + 4 * b + r;
                            const bool hide = (flags >> (2 * h) & 2) || k < lo[t] || k > hi[t];
                            s[t][h][r] = hide ? -INFINITY : s[t][h][r];
                            hidden[t] |= hide ? 1u << (4 * h + at_place(r)) : 0u;
                        }
                }
            } else if (flags) {
#pragma unroll
                for (int t = 0; t < NT; t++) hidden[t] = 0;
            }
            float top[NT];
            bool more = false;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                top[t] = s[t][0][0];
#pragma unroll
                for (int x = 1; x < 8; x++) top[t] = fmaxf(top[t], s[t][x >> 2][x & 3]);
                top[t] *= fac[t];
                more |= top[t] > m[t] + AT_SLACK;
            }
            if (__any(more)) {
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const float to = fmaxf(m[t], at_max4(top[t])), f = to == -INFINITY ? 1.0f : at_exp2(m[t] - to);
                    m[t] = to;
                    l[t] *= f;
#pragma unroll
                    for (int j = 0; j < 2 * G; j++) o[t][j] *= f;
                }
            }
            kv_h8 pf[NT][PARTS];
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const float off = AT_P2 - (m[t] == -INFINITY ? 0.0f : m[t]);
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    const int h = x >> 2, r = x & 3, at = 4 * h + at_place(r);
                    const float p = at_exp2(fmaf(s[t][h][r], fac[t], off));
                    pf[t][0][at] = (_Float16)p;
                    if constexpr (PARTS == 2) pf[t][1][at] = (_Float16)(p - (float)pf[t][0][at]);
                }
            }
#pragma unroll
            for (int j = 0; j < 2 * G; j++) {
                const kv_h8 a = sh.v[buf][blk][j][lane];
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int p = 0; p < PARTS; p++) o[t][j] = at_mfma(a, pf[t][p], o[t][j]);
            }
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int p = 0; p < PARTS; p++) l[t] = at_mfma(ones, pf[t][p], l[t]);
            if (flags & 5) {                             // how many NaN a row sees, for each of its values
                asm volatile("");
#pragma unroll
                for (int j = 0; j < 2 * G; j++) {
                    const int g = (2 * G * col + j) >> 5;
                    uint32_t bits = 0;
                    if (flags & 1) bits |= sh.nan[buf][2 * blk][g] >> (4 * b) & 15;
                    if (flags & 4) bits |= (sh.nan[buf][2 * blk + 1][g] >> (4 * b) & 15) << 4;
                    const kv_h8 a = at_ones(bits);
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const kv_f4 n = at_mfma(a, at_ones(~hidden[t]), kv_f4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (n[i] > 0.0f) o[t][j][i] = NAN;
                    }
                }
            }
        };

        __syncthreads();                                 // the block before this one has been read
        int buf = 0;
        if (st < st1) {
            convert(0, key_of(st), pg);
            pg = pn;
            pn = entry(key_of(st + 2));
            if (st + 1 < st1) load(key_of(st + 1), pg);
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma clang loop unroll(disable)
        for (; st < st1; st++, buf ^= 1) {
            if (st + 1 < st1) {
                convert(buf ^ 1, key_of(st + 1), pg);
                pg = pn;
                pn = entry(key_of(st + 3));
                if (st + 2 < st1) load(key_of(st + 2), pg);
            }
            const int key = key0 + st * ST;
#pragma unroll
            for (int blk = 0; blk < 2; blk++)
                if (key + 32 * blk <= hi_max && key + 32 * blk + 31 >= lo_min) work(buf, blk, key + 32 * blk);
            // LDS writes are done; loads that are on their way end in registers, which their uses wait for
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int r = row0 + 16 * t + col;
            if (r >= rows) continue;
            const int i = r / L.g, h = it.head * L.g + r - i * L.g;
            const float sum = l[t][0];
            if (parts > 1) {
                float *const to = prompt_piece<D, RB>(P, it.item, it.part);
                const int rr = r - block * RB;
                if (b == 0) { to[RB * D + rr] = m[t]; to[RB * D + RB + rr] = sum; }
#pragma unroll
                for (int x = 0; x < 4; x++)
#pragma unroll
                    for (int j = 0; j < 2 * G; j += 2) {
                        typedef float f2 __attribute__((ext_vector_type(2)));
                        *(f2 *)(to + rr * D + 2 * G * (4 * b + x) + j) = f2{o[t][j][x], o[t][j + 1][x]};
                    }
                continue;
            }
            const float f = attn_factor(m[t], sum, L.a.sink != nullptr, L.a.sink ? L.a.sink[h] * 1.44269504088896340736f : 0.0f);
            const long at = (long)(q.begin + i) * L.a.ldo + (long)h * L.a.hdo;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const long d = at + 2 * G * (4 * b + x);
                if constexpr (G % 4 == 0) {
#pragma unroll
                    for (int j = 0; j < 2 * G; j += 8) {
                        float y[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) y[e] = o[t][j + e][x] * f;
                        kv_store8(L.a.out, L.a.type, d + j, y);
                    }
                } else if constexpr (G % 2 == 0) {
#pragma unroll
                    for (int j = 0; j < 2 * G; j += 4) kv_store4(L.a.out, L.a.type, d + j, kv_f4{o[t][j][x], o[t][j + 1][x], o[t][j + 2][x], o[t][j + 3][x]} * f);
                } else {
#pragma unroll
                    for (int j = 0; j < 2 * G; j++) i8_st(L.a.out, L.a.type, (size_t)(d + j), o[t][j][x] * f);
                }
            }
        }
    }
}

// The parts of split blocks: 256 threads for 256 / (D / 4) rows of an item at a time.
template <int D, int RB>
__global__ __launch_bounds__(256) void k_attn_join(PromptLaunch P) {
    const AttnLaunch &L = P.A;
    long x = blockIdx.x;
    const int head = (int)(x % L.c.heads), s = (int)(x / L.c.heads % L.a.S), block = (int)(x / L.c.heads / L.a.S);
    const AttnSeq q = attn_seq(L, s);
    if ((long)q.n * L.g <= L.limit) return;
    const int r = (int)blockIdx.y * (256 / (D / 4)) + (int)threadIdx.x / (D / 4), d = (int)threadIdx.x % (D / 4) * 4;
    if (r >= RB || (int)threadIdx.x >= 256 / (D / 4) * (D / 4) || block * RB + r >= q.n * L.g) return;
    float M = -INFINITY, sum = 0.0f;
    for (int p = 0; p < P.parts; p++) M = fmaxf(M, prompt_piece<D, RB>(P, x, p)[RB * D + r]);
    kv_f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int p = 0; p < P.parts; p++) {
        const float *const at = prompt_piece<D, RB>(P, x, p);
        const float m = at[RB * D + r], f = m == -INFINITY ? 0.0f : at_exp2(m - M);
        v += *(const kv_f4 *)(at + r * D + d) * f;
        sum += at[RB * D + RB + r] * f;
    }
    const int i = (block * RB + r) / L.g, h = head * L.g + (block * RB + r) - i * L.g;
    v *= attn_factor(M, sum, L.a.sink != nullptr, L.a.sink ? L.a.sink[h] * 1.44269504088896340736f : 0.0f);
    kv_store4(L.a.out, L.a.type, (long)(q.begin + i) * L.a.ldo + (long)h * L.a.hdo + d, v);
}

// ================================================================================== host side
template <int G, int WAVES, int NT, int PARTS>
static int prompt_go(bgl_ctx *c, const AttnLaunch &L) {
    constexpr int RB = 16 * NT * WAVES, D = 32 * G;
    PromptLaunch P;
    memset(&P, 0, sizeof P);
    P.A = L;
    const long rows = (long)std::min(std::max(1, L.a.max_rows), L.a.T) * L.g;
    P.blocks = (int)((rows + RB - 1) / RB);
    const long items = (long)P.blocks * L.a.S * L.c.heads;
    // few blocks: their keys in parts, of 256 keys at least
    const int at_once = WAVES == 8 ? 256 : 512;
    P.parts = (int)std::max<long>(1, std::min<long>({16, at_once / std::max(1l, items), ((long)std::max(1, L.a.max_len) + 255) / 256}));
    if (items * P.parts > INT32_MAX / 4) return bgl_fail(BGL_E_ARG, "bgl_attn_dev: %d sequences of up to %d rows", L.a.S, L.a.max_rows);
    if (P.parts > 1) {
        if (const int rc = dbuf_reserve(c, c->attn_part, (size_t)items * P.parts * RB * (D + 2) * 4, false)) return rc;
        P.A.part = (float *)c->attn_part.p;
    }
    hipLaunchKernelGGL((k_attn_prompt<G, WAVES, NT, PARTS>), dim3((unsigned)(items * P.parts)), dim3(64 * WAVES), 0, c->stream, P);
    if (P.parts > 1) {
        constexpr int per = 256 / (D / 4);
        hipLaunchKernelGGL((k_attn_join<D, RB>), dim3((unsigned)items, (RB + per - 1) / per), dim3(256), 0, c->stream, P);
    }
    return 0;
}
template <int G>
static int prompt_pick(bgl_ctx *c, const AttnLaunch &L) {
    if (L.a.type == BGL_T_F32) return prompt_go<G, 8, G <= 4 ? 2 : 1, 2>(c, L);
    return prompt_go<G, 8, G <= 6 ? 2 : 1, 1>(c, L);
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
