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

template <int G, int NT, int PARTS>
struct Prompt {
    static constexpr int D = 32 * G, WAVES = 8, RB = 16 * NT * WAVES, ST = 64;
    static constexpr bool K2 = G % 3 == 0 || G > 4, V2 = G % 3 == 0;                  // as in AttnRaw
    struct Shared {
        kv_h8 k[2][4][G][64], v[2][2][2 * G][64];
        at_u4 flag[2];                                   // a tile each: 1 some value of V is NaN, 2 it has no page
    };
};

template <int G, int NT, int PARTS>
__global__ __launch_bounds__(512, 2) void k_attn_prompt(PromptLaunch P) {
    using T = Prompt<G, NT, PARTS>;
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
    // In the loop over keys the table is read by vector loads: a scalar load on its way makes every wait for the LDS a wait for all of it.
    const int *vtable = L.a.table + (size_t)it.s * L.a.ldt;
    int zero_lane = 0;
    asm volatile("" : "+v"(zero_lane));
    const int last_page = at_page(L, max(0, q.len - 1) >> 4);
    // A wave converts, of each stage's four tiles, K or V of one.
    const int tile = wave >> 1;
    const bool of_v = wave & 1;
    const int codes_at = (of_v ? 10 * D : 0) + lane * (4 * G);
    const int steps_at = of_v ? 18 * D + ((G * col >> 4) * 4 + b) * 16 : 8 * D + ((G * b >> 2) * 16 + col) * 4;
    const int steps_at2 = of_v ? 18 * D + (((G * col + G - 1) >> 4) * 4 + b) * 16 : 8 * D + (((G * b + G - 1) >> 2) * 16 + col) * 4;
    for (int block = it.block; block * RB < rows; block += P.blocks) {
        // the keys of the block's rows, this part's stages of 64 among them
        int lo_first, lo_last, hi_first, hi_last;
        attn_keys(L, q, block * RB / L.g, lo_first, hi_first);
        attn_keys(L, q, (min(block * RB + RB, rows) - 1) / L.g, lo_last, hi_last);
        const int key0 = lo_first & ~15, stages = max(0, (hi_last + 1 - key0 + ST - 1) / ST);
        const int parts = block < P.blocks ? P.parts : 1;          // blocks that max_rows did not tell of have no room for pieces
        if (it.part >= parts) break;
        const int st0 = __builtin_amdgcn_readfirstlane((int)((long)stages * it.part / parts));
        const int st1 = __builtin_amdgcn_readfirstlane((int)((long)stages * (it.part + 1) / parts));

        auto key_of = [&](int stage) { return key0 + stage * ST + 16 * tile; };
        auto entry = [&](int stage) { return vtable[min(at_page(L, key_of(stage) >> 4), last_page) + zero_lane]; };
        auto page = [&](int stage, int e) {              // the page, or -1: past the keys, or none
            e = __builtin_amdgcn_readfirstlane(e);
            return key_of(stage) < q.len && (uint32_t)e < (uint32_t)L.c.pages ? e : -1;
        };
        uint32_t codes[G];
        typedef unsigned int u4 __attribute__((ext_vector_type(4), aligned(4)));
        at_u4 steps, steps2;
        // (a tile without a page loads the first record, and none of it counts)
        auto load = [&](int stage, int pg) {
            const int t = key_of(stage) >> 4;
            const size_t rec = pg < 0 ? 0 : ((size_t)pg * L.c.heads + it.head) * L.ppt + (t - at_page(L, t) * L.ppt);
            const uint8_t *p = (const uint8_t *)L.c.data + rec * (20 * D);
            at_dwords<G>(codes, p + codes_at);
            steps = *(const u4 *)(p + steps_at);
            if constexpr (K2 || V2) steps2 = *(const u4 *)(p + steps_at2);
        };
        auto convert = [&](int buf, int stage, int pg) {
            if (!of_v) {
#pragma unroll
                for (int j = 0; j < G; j++)
                    sh.k[buf][tile][j][lane] = at_key(magic, codes[j], K2 && (G * b + j) >> 2 != G * b >> 2 ? steps2[0] : steps[0]);
                return;
            }
            uint32_t flag = pg < 0 ? 2 : 0;
            if (pg < 0 || key_of(stage) + 16 > q.len) {  // what lies behind the last key may be anything: 0
                asm volatile("");
                const int left = pg < 0 ? 0 : q.len - key_of(stage) - 4 * b;           // of the lane's four keys
                const uint32_t e = (left > 0 ? 0x0000ffffu : 0u) | (left > 2 ? 0xffff0000u : 0u);
                const uint32_t f = (left > 1 ? 0x0000ffffu : 0u) | (left > 3 ? 0xffff0000u : 0u);
                steps &= at_u4{e, f, e, f};
                if constexpr (V2) steps2 &= at_u4{e, f, e, f};
            }
            bool nan = at_clean(steps);
            if constexpr (V2) nan |= at_clean(steps2);
            if (__any(nan)) flag |= 1;
#pragma unroll
            for (int j = 0; j < G; j++) {
                const at_u4 z = V2 && (G * col + j) >> 4 != G * col >> 4 ? steps2 : steps;
                const kv_h2 s0 = __builtin_bit_cast(kv_h2, (uint32_t)z[0]), s1 = __builtin_bit_cast(kv_h2, (uint32_t)z[1]);
                const kv_h2 m0 = __builtin_bit_cast(kv_h2, (uint32_t)z[2]), m1 = __builtin_bit_cast(kv_h2, (uint32_t)z[3]);
                const uint32_t c = codes[j], d = c >> 8;
                typedef uint32_t u2 __attribute__((ext_vector_type(2)));
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    u2 w;
                    w[0] = __builtin_bit_cast(uint32_t, e ? at_hi(magic, c, s0, m0) : at_lo(magic, c, s0, m0));
                    w[1] = __builtin_bit_cast(uint32_t, e ? at_hi(magic, d, s1, m1) : at_lo(magic, d, s1, m1));
                    ((u2 *)&sh.v[buf][tile >> 1][2 * j + e][lane])[tile & 1] = w;
                }
            }
            if (lane == 0) ((uint32_t *)&sh.flag[buf])[tile] = flag;
        };

        int pg = page(st0, entry(st0));
        load(st0, pg);
        int next = entry(st0 + 1);
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

        bool nan = false;                                // V has had one
        // A stage's operands in runs of G, each read from the LDS while the run before it is multiplied: K of tiles 0 .. 3, then V of
        // both halves, values 0 .. G - 1 and G .. 2 G - 1.
        kv_h8 f[2][G];
        auto read = [&](int buf, int run) {
#pragma unroll
            for (int j = 0; j < G; j++) f[run & 1][j] = run < 4 ? sh.k[buf][run][j][lane] : sh.v[buf][(run - 4) >> 1][((run & 1) ? G : 0) + j][lane];
        };
        auto work = [&](int buf, int key) {
            const at_u4 fl = sh.flag[buf];
            kv_f4 s[NT][4];
#pragma unroll
            for (int h = 0; h < 4; h++) {
                read(buf, h + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < G; j++)
#pragma unroll
                    for (int p = 0; p < PARTS; p++)
#pragma unroll
                        for (int t = 0; t < NT; t++)
                            s[t][h] = at_mfma(f[h & 1][j], qf[t][p][j], j + p ? s[t][h] : kv_f4{zero[t], zero[t], zero[t], zero[t]});
            }
            const uint32_t flags = (uint32_t)__builtin_amdgcn_readfirstlane((int)(fl[0] | fl[1] << 2 | fl[2] << 4 | fl[3] << 6));
            if ((flags & 0xaa) || key < lo_max || key + ST - 1 > hi_min) {
                asm volatile("");
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const int from = at_from(lo[t], key + 4 * b), to = at_from(hi[t], key + 4 * b);
#pragma unroll
                    for (int h = 0; h < 4; h++) {
                        const int last = flags >> (2 * h) & 2 ? -1 : to;               // no page
#pragma unroll
                        for (int r = 0; r < 4; r++) s[t][h][r] = at_hide(s[t][h][r], at_hides(16 * h + r, from, last));
                    }
                }
            }
            float top[NT];
            bool more = false;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                top[t] = s[t][0][0];
#pragma unroll
                for (int x = 1; x < 16; x++) top[t] = fmaxf(top[t], s[t][x >> 2][x & 3]);
                top[t] *= fac[t];
                more |= top[t] > m[t] + AT_SLACK;
            }
            if (__any(more)) {
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const float to = fmaxf(m[t], at_max4(top[t])), g = to == -INFINITY ? 1.0f : at_exp2(m[t] - to);
                    m[t] = to;
                    l[t] *= g;
#pragma unroll
                    for (int j = 0; j < 2 * G; j++) o[t][j] *= g;
                }
            }
            kv_h8 pf[2][NT][PARTS];
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const float off = AT_P2 - (m[t] == -INFINITY ? 0.0f : m[t]);
#pragma unroll
                for (int x = 0; x < 16; x++) {
                    const int h = x >> 2, r = x & 3, at = 4 * (h & 1) + at_place(r);
                    const float p = at_exp2(fmaf(s[t][h][r], fac[t], off));
                    pf[h >> 1][t][0][at] = (_Float16)p;
                    if constexpr (PARTS == 2) pf[h >> 1][t][1][at] = (_Float16)(p - (float)pf[h >> 1][t][0][at]);
                }
            }
#pragma unroll
            for (int run = 4; run < 8; run++) {
                const int i = (run - 4) >> 1;
                if (run < 7) read(buf, run + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < G; j++)
#pragma unroll
                    for (int p = 0; p < PARTS; p++)
#pragma unroll
                        for (int t = 0; t < NT; t++) o[t][(run & 1) * G + j] = at_mfma(f[run & 1][j], pf[i][t][p], o[t][(run & 1) * G + j]);
                if (run & 1) {
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int p = 0; p < PARTS; p++) l[t] = at_mfma(ones, pf[i][t][p], l[t]);
                }
            }
            if (flags & 0x55) nan = true;
        };

        __syncthreads();                                 // the block before this one has been read
        convert(0, st0, pg);                             // (without a stage: of a tile past the keys, or one that nothing reads)
        int pn = page(st0 + 1, next);
        load(st0 + 1, pn);
        next = entry(st0 + 2);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        int buf = 0;
#pragma clang loop unroll(disable)
        for (int st = st0; st < st1; st++, buf ^= 1) {
            const int key = key0 + st * ST;
            const bool mine = key <= hi_max && key + ST - 1 >= lo_min;
            if (mine) read(buf, 0);
            __builtin_amdgcn_sched_barrier(0);
            convert(buf ^ 1, st + 1, pn);
            pn = page(st + 2, next);
            load(st + 2, pn);
            next = entry(st + 3);
            __builtin_amdgcn_sched_barrier(0);
            if (mine) work(buf, key);
            // LDS writes are done; loads that are on their way end in registers, which their uses wait for
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        if (nan)
            for (int key = key0 + st0 * ST; key < key0 + st1 * ST; key += 32) at_nan<G, NT>(L, q, it.head, table, key, lane, lo, hi, o);
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
template <int G, int NT, int PARTS>
static int prompt_go(bgl_ctx *c, const AttnLaunch &L) {
    constexpr int RB = Prompt<G, NT, PARTS>::RB, D = 32 * G;
    PromptLaunch P;
    memset(&P, 0, sizeof P);
    P.A = L;
    const long rows = (long)std::min(std::max(1, L.a.max_rows), L.a.T) * L.g;
    P.blocks = (int)((rows + RB - 1) / RB);
    const long items = (long)P.blocks * L.a.S * L.c.heads;
    // few blocks: their keys in parts, of 256 keys at least
    const int at_once = 256;
    P.parts = (int)std::max<long>(1, std::min<long>({16, at_once / std::max(1l, items), ((long)std::max(1, L.a.max_len) + 255) / 256}));
    if (items * P.parts > INT32_MAX / 4) return bgl_fail(BGL_E_ARG, "bgl_attn_dev: %d sequences of up to %d rows", L.a.S, L.a.max_rows);
    if (P.parts > 1) {
        if (const int rc = dbuf_reserve(c, c->attn_part, (size_t)items * P.parts * RB * (D + 2) * 4, false)) return rc;
        P.A.part = (float *)c->attn_part.p;
    }
    hipLaunchKernelGGL((k_attn_prompt<G, NT, PARTS>), dim3((unsigned)(items * P.parts)), dim3(512), 0, c->stream, P);
    if (P.parts > 1) {
        constexpr int per = 256 / (D / 4);
        hipLaunchKernelGGL((k_attn_join<D, RB>), dim3((unsigned)items, (RB + per - 1) / per), dim3(256), 0, c->stream, P);
    }
    return 0;
}
template <int G>
static int prompt_pick(bgl_ctx *c, const AttnLaunch &L) {
    if (L.a.type == BGL_T_F32) return prompt_go<G, G <= 4 ? 2 : 1, 2>(c, L);
    return prompt_go<G, G <= 4 ? 2 : 1, 1>(c, L);
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
