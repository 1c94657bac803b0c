// bgl_attn.hip -- attention of a few rows a sequence (single tokens, drafted ones) over the paged cache in 4 bits:
//
//   s_j = scale q . k_j;   out = sum_j exp(s_j - M) v_j / sum_j exp(s_j - M)      one pass: M, both sums and out run along
//
// The rows are bound by the cache's bytes, 1.25 D for a key and head, read once for all of a head's group of query rows.  Those
// rows (g heads of q times the tokens) are the 16 columns of the matrix instruction, keys its rows:
//   scores   S^T = K Q^T: a lane has 4 keys of one query row from each 16-key tile
//   output   O^T = V^T P^T: what a lane has of S^T is, as weights, its part of P^T's operand: nothing is moved between lanes
// but the row maxima; a row's statistics lie in the lanes that hold its sums.
//
// Work: 128 keys of one head and row block are a unit, 32 for each wave (or 512, where no sequence has more).  The units of all
// sequences lie in one line (short sequences apart, attn_pause) that is cut into equal runs, one a workgroup, so a batch of very
// different lengths leaves no workgroup behind.  A head whose keys end up in several runs is joined by whichever of them
// finishes last, in the order of its keys: the same bits every time.
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

#define AT_STEP 128              // keys that the four waves of a workgroup go over at once
#define AT_WG 512                // workgroups at most: two for each CU, so that all run at once (three, where registers allow it: 31.6 us for 30.0)
#define AT_FEW 32                // rows of a head's group that a sequence of few rows has, at most
#define AT_SC1 16                // the cache-policy bit of a buffer access of device scope

// What a wave has loaded of 32 keys: two tiles.
template <int G>
struct AttnRaw {
    static constexpr bool K2 = G % 3 == 0 || G > 4, V2 = G % 3 == 0;      // a lane's values lie in one group of 32, or in two
    uint32_t kc[2][G], vc[2][G], ks[2][K2 ? 2 : 1];
    at_u4 vs[2][V2 ? 2 : 1];
};

template <int G, int NT, int PARTS>
struct AttnWave {
    static constexpr int D = 32 * G, RB = 16 * NT;
    const AttnLaunch &L;
    const int lane, col, b;                              // col: the lane's query row of each 16, key of a K tile, unit of a V tile
    AttnSeq q;
    int head;
    ucint table;
    const AtMagic magic;
    AtQuery<G, PARTS> query[NT];
    kv_h8 qf[NT][1][PARTS][G];
    float fac[NT], zero[NT];                             // zero: where scores begin; NaN for a query with a NaN or an infinity
    int lo[NT], hi[NT], lo_max, hi_min;
    kv_f4 o[NT][2 * G];
    float m[NT], l[NT];
    bool nan;                                            // V has had one, in a lane's keys

    __device__ AttnWave(const AttnLaunch &l_) : L(l_), lane(threadIdx.x & 63), col(threadIdx.x & 15), b((threadIdx.x >> 4) & 3) {}

    // Rows rb * RB .. of the sequence's n * g: their loads, then their operands.
    __device__ __forceinline__ void ask(int rb) {
#pragma unroll
        for (int t = 0; t < NT; t++) query[t].load(L, q, head, rb * RB + 16 * t + col, b);
    }
    __device__ __forceinline__ void begin(int rb) {
        lo_max = 0;
        hi_min = INT32_MAX;
        nan = false;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            query[t].operands(L, qf[t], fac[t], zero[t]);
            attn_keys(L, q, min(rb * RB + 16 * t + col, q.n * L.g - 1) / L.g, lo[t], hi[t]);
            lo_max = max(lo_max, lo[t]);
            hi_min = min(hi_min, hi[t]);
            m[t] = -INFINITY;
            l[t] = 0.0f;
#pragma unroll
            for (int j = 0; j < 2 * G; j++) o[t][j] = kv_f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        lo_max = -at_min16(-lo_max);
        hi_min = at_min16(hi_min);
    }

    // The table's entry for the tile at a key (a multiple of 16); -1 past the keys.  It may name no page.
    __device__ __forceinline__ int entry(int key) const { return key < q.len ? table[at_page(L, key >> 4)] : -1; }
    // The record of the tile at a key, in the page of the table's entry; a tile without a page loads the first record, and none of
    // it counts.
    __device__ __forceinline__ const uint8_t *record(int key, int pg) const {
        const int t = key >> 4;
        const size_t rec = none(pg) ? 0 : ((size_t)pg * L.c.heads + head) * L.ppt + (t - at_page(L, t) * L.ppt);
        return (const uint8_t *)L.c.data + rec * (20 * D);
    }
    __device__ __forceinline__ void load_k(AttnRaw<G> &w, int h, const uint8_t *p) const {
        at_dwords<G>(w.kc[h], p + lane * (4 * G));
        const uint32_t *ks = (const uint32_t *)(p + 8 * D);
        w.ks[h][0] = ks[(G * b >> 2) * 16 + col];
        if constexpr (AttnRaw<G>::K2) w.ks[h][1] = ks[((G * b + G - 1) >> 2) * 16 + col];
    }
    __device__ __forceinline__ void load_v(AttnRaw<G> &w, int h, const uint8_t *p) const {
        at_dwords<G>(w.vc[h], p + 10 * D + lane * (4 * G));
        const at_u4 *vs = (const at_u4 *)(p + 18 * D);
        w.vs[h][0] = vs[(G * col >> 4) * 4 + b];
        if constexpr (AttnRaw<G>::V2) w.vs[h][1] = vs[((G * col + G - 1) >> 4) * 4 + b];
    }
    __device__ __forceinline__ bool none(int pg) const { return (uint32_t)pg >= (uint32_t)L.c.pages; }

    // Keys key .. key + 31 into m, l and o.  next: the records of the wave's next 32 keys, or null; they are loaded into the registers
    // that this step has used up.
    __device__ __forceinline__ void step(AttnRaw<G> &w, int key, const int (&pg)[2], const uint8_t *const (&next)[2]) {
        constexpr bool K2 = AttnRaw<G>::K2, V2 = AttnRaw<G>::V2;
        kv_f4 s[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++) s[t][0] = s[t][1] = kv_f4{zero[t], zero[t], zero[t], zero[t]};
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int j = 0; j < G; j++) {
                const uint32_t sm = K2 && (G * b + j) >> 2 != G * b >> 2 ? w.ks[h][K2] : w.ks[h][0];
                const kv_h8 k = at_key(magic, w.kc[h][j], sm);
#pragma unroll
                for (int t = 0; t < NT; t++) {
#pragma unroll
                    for (int p = 0; p < PARTS; p++) s[t][h] = at_mfma(k, qf[t][0][p][j], s[t][h]);
                }
            }
        }
        if (next[0]) {
            load_k(w, 0, next[0]);
            load_k(w, 1, next[1]);
        }
        // Some of the keys may be hidden from some rows: at the last key, along the rows' diagonal, at the window's edge.  (The empty
        // asm keeps the compiler from doing this for every unit, with selects.)
        if (none(pg[0]) || none(pg[1]) || key < lo_max || key + 31 > hi_min) {
            asm volatile("");
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int k0 = key + 16 * h + 4 * b;
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const int from = at_from(lo[t], k0), to = none(pg[h]) ? -1 : at_from(hi[t], k0);
#pragma unroll
                    for (int r = 0; r < 4; r++) s[t][h][r] = at_hide(s[t][h][r], at_hides(r, from, to));
                }
                // Memory behind the last key holds anything: 0 there, which a weight of 0 leaves 0.
                const int left = none(pg[h]) ? 0 : q.len - k0;
                const uint32_t e = (left > 0 ? 0x0000ffffu : 0u) | (left > 2 ? 0xffff0000u : 0u);
                const uint32_t f = (left > 1 ? 0x0000ffffu : 0u) | (left > 3 ? 0xffff0000u : 0u);
#pragma unroll
                for (int x = 0; x < (V2 ? 2 : 1); x++) {
                    w.vs[h][x] &= at_u4{e, f, e, f};
                    nan |= at_clean(w.vs[h][x]);
                }
            }
        }
        kv_h8 pf[NT][PARTS];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            float top = s[t][0][0];
#pragma unroll
            for (int x = 1; x < 8; x++) top = fmaxf(top, s[t][x >> 2][x & 3]);
            top *= fac[t];
            if (__any(top > m[t] + AT_SLACK)) {
                const float to = fmaxf(m[t], at_max4(top)), f = to == -INFINITY ? 1.0f : at_exp2(m[t] - to);
                m[t] = to;
                l[t] *= f;
#pragma unroll
                for (int j = 0; j < 2 * G; j++) o[t][j] *= f;
            }
            const float off = AT_P2 - (m[t] == -INFINITY ? 0.0f : m[t]);
#pragma unroll
            for (int x = 0; x < 8; x++) {
                const int h = x >> 2, r = x & 3;
                const float p = at_exp2(fmaf(s[t][h][r], fac[t], off));
                if constexpr (PARTS == 2) l[t] += p;
                const int at = 4 * h + at_place(r);
                pf[t][0][at] = (_Float16)p;
                if constexpr (PARTS == 2) pf[t][1][at] = (_Float16)(p - (float)pf[t][0][at]);
            }
            // One fp16 part of the weights for 16-bit rows: 2^-11 of each, which an average of many keys makes less of (error against 64 bits: fp16
            // rows 2.4e-4 for the 2.1e-4 of the output's own rounding, bf16 rows 1.7e-3 either way).  A second part costs 28.8 -> 30.2 us (32 sequences of 111 to 8192
            // keys), 40.8 -> 43.1 (131072 keys), in the prompt kernel 41 -> 51 (chunks of 9 sequences) and 160 -> 229 (4096 tokens).
            // Weights rounded to fp16 are summed as what they are multiplied as, so that a row's add up to 1: their error is then that of an average
            // of values (unrounded sums: a row whose keys all have the value v was up to 4e-4 v off).  Two parts are 2^-22 off p.
            if constexpr (PARTS == 1) {
                const kv_h2 one = {(_Float16)1.0f, (_Float16)1.0f};
                float sum[2] = {0.0f, 0.0f};
#pragma unroll
                for (int y = 0; y < 8; y += 2) sum[y >> 2] = __builtin_amdgcn_fdot2(kv_h2{pf[t][0][y], pf[t][0][y + 1]}, one, sum[y >> 2], false);
                l[t] += sum[0] + sum[1];
            }
        }
#pragma unroll
        for (int j = 0; j < G; j++) {
            kv_h2 v[2][4];                               // values 2 j (pairs 0, 2 and 1, 3 of each tile) and 2 j + 1
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const at_u4 z = V2 && (G * col + j) >> 4 != G * col >> 4 ? w.vs[h][V2] : w.vs[h][0];
                const kv_h2 s0 = __builtin_bit_cast(kv_h2, (uint32_t)z[0]), s1 = __builtin_bit_cast(kv_h2, (uint32_t)z[1]);
                const kv_h2 m0 = __builtin_bit_cast(kv_h2, (uint32_t)z[2]), m1 = __builtin_bit_cast(kv_h2, (uint32_t)z[3]);
                const uint32_t c = w.vc[h][j], d = c >> 8;
                v[0][2 * h] = at_lo(magic, c, s0, m0);
                v[0][2 * h + 1] = at_lo(magic, d, s1, m1);
                v[1][2 * h] = at_hi(magic, c, s0, m0);
                v[1][2 * h + 1] = at_hi(magic, d, s1, m1);
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const kv_h8 a = at_join(v[e][0], v[e][1], v[e][2], v[e][3]);
#pragma unroll
                for (int t = 0; t < NT; t++) {
#pragma unroll
                    for (int p = 0; p < PARTS; p++) o[t][2 * j + e] = at_mfma(a, pf[t][p], o[t][2 * j + e]);
                }
            }
        }
        if (next[0]) {
            load_v(w, 0, next[0]);
            load_v(w, 1, next[1]);
        }
    }
};

#define AT_JOIN 32               // pieces that are joined at once, at most
template <int G, int NT>
struct AttnShared {
    static constexpr int D = 32 * G, RB = 16 * NT, ROW = D + 4;
    float m[4][RB], l[4][RB], M[RB], sum[RB];
    int last;
    union {
        float o[4][RB][ROW];
        struct { float m[AT_JOIN][RB], l[AT_JOIN][RB]; } j;
    };
};

// A sequence's row blocks and, for each of them and a head (an item), the units of keys.
template <int RB>
__device__ __forceinline__ void attn_units(const AttnLaunch &L, const AttnSeq &q, int &blocks, int &chunks) {
    blocks = q.n > 0 && (long)q.n * L.g <= L.limit ? (q.n * L.g + RB - 1) / RB : 0;
    chunks = max(1, (q.len - (q.lo & ~15) + L.unit - 1) / L.unit);
}
// Starting and ending an item takes a workgroup as long as one to three units, the more the more of memory's rate each workgroup has.  Items
// shorter than a run lie that far apart in the line, or the workgroups that have the short sequences would be the last (8 heads, 32 sequences of 111 to
// 8192 keys: 38.6 us without pauses, 28.5 with one unit, 29.4 with two; 200 of 200 to 3000 keys: 96, 83, 77, 75 with three; 32 of 2048 keys each 23.5).
#define AT_PAUSE 3
__device__ __forceinline__ int attn_pause(int chunks, int run) { return chunks < run ? min(max(run >> 3, 1), AT_PAUSE) : 0; }

// The line of units in runs: the first `more` workgroups have one unit more than the others' `each`.
struct AttnRuns {
    uint32_t each, more, wgs;
    __device__ AttnRuns(uint32_t total, uint32_t grid, uint32_t least) {
        wgs = min(grid, total < 64 ? total : (total + least - 1) / least);
        each = wgs ? total / wgs : 0;
        more = total - each * wgs;
    }
    __device__ __forceinline__ uint32_t begin(uint32_t w) const { return w * each + min(w, more); }
    __device__ __forceinline__ uint32_t owner(uint32_t u) const {
        const uint32_t head = more * (each + 1);
        return u < head ? u / (each + 1) : more + (u - head) / each;
    }
};

template <int G, int NT, int PARTS>
__global__ __launch_bounds__(256, 2) void k_attn(AttnLaunch L) {
    using Wave = AttnWave<G, NT, PARTS>;
    constexpr int D = 32 * G, RB = 16 * NT, PIECE = RB * (D + 2);
    __shared__ AttnShared<G, NT> sh;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), heads = L.c.heads, S = L.a.S;
    // Every wave counts all units by itself, lane by lane, each lane `per` sequences.
    const int per = (S + 63) / 64, lane = tid & 63;
    AttnSeq mine_q;
    mine_q.begin = mine_q.n = mine_q.len = mine_q.lo = 0;
    int mine = 0;
    bool back = false;                                   // starts go back: the units could be more than the host has checked for
    for (int s = lane * per; s < min(S, (lane + 1) * per); s++) {
        int blocks, chunks;
        mine_q = attn_seq(L, s);
        attn_units<RB>(L, mine_q, blocks, chunks);
        mine += blocks * heads * chunks;
        back |= min(L.a.start[s + 1], L.a.T) < mine_q.begin;
    }
    if (__any(back)) return;
    int upto = at_scan(mine);                            // units up to the end of the lane's sequences
    const int run = (int)((uint32_t)__builtin_amdgcn_readlane(upto, 63) / gridDim.x);            // without pauses
    if (run > 1) {
        mine = 0;
        for (int s = lane * per; s < min(S, (lane + 1) * per); s++) {
            int blocks, chunks;
            if (per > 1) mine_q = attn_seq(L, s);
            attn_units<RB>(L, mine_q, blocks, chunks);
            mine += blocks * heads * (chunks + attn_pause(chunks, run));
        }
        upto = at_scan(mine);
    }
    const __amdgpu_buffer_rsrc_t pieces = __builtin_amdgcn_make_buffer_rsrc(L.part, (short)0, AT_WG * 2 * PIECE * 4, 0x00020000);
    const AttnRuns runs((uint32_t)__builtin_amdgcn_readlane(upto, 63), gridDim.x, (uint32_t)L.least);
    const uint32_t w = blockIdx.x;
    if (w >= runs.wgs) return;
    const uint32_t end = runs.begin(w + 1);
    uint32_t u = runs.begin(w);
    Wave W(L);
    int blocks, chunks;
    while (u < end) {
        // the sequence of unit u: the first lane whose sequences end behind it, then that lane's sequences in turn
        const int at_lane = __popcll(__ballot((uint32_t)upto <= u));
        uint32_t base = (uint32_t)__builtin_amdgcn_readlane(upto - mine, at_lane);     // units before sequence s
        int s = at_lane * per;
        W.q.begin = __builtin_amdgcn_readlane(mine_q.begin, at_lane);
        W.q.n = __builtin_amdgcn_readlane(mine_q.n, at_lane);
        W.q.len = __builtin_amdgcn_readlane(mine_q.len, at_lane);
        W.q.lo = __builtin_amdgcn_readlane(mine_q.lo, at_lane);
        attn_units<RB>(L, W.q, blocks, chunks);
        if (per > 1) {
            while (true) {
                W.q = attn_seq(L, s);
                W.q.begin = __builtin_amdgcn_readfirstlane(W.q.begin);
                W.q.n = __builtin_amdgcn_readfirstlane(W.q.n);
                W.q.len = __builtin_amdgcn_readfirstlane(W.q.len);
                W.q.lo = __builtin_amdgcn_readfirstlane(W.q.lo);
                attn_units<RB>(L, W.q, blocks, chunks);
                const uint32_t n = (uint32_t)(blocks * heads * (chunks + attn_pause(chunks, run)));
                if (u < base + n) break;
                base += n;
                s++;
            }
        }
        const int pause = attn_pause(chunks, run), span = chunks + pause;
        const int item = (int)((u - base) / (uint32_t)span);                         // head * blocks + row block
        const int head = item / blocks, rb = item - head * blocks;
        const int at = (int)(u - base) - item * span;    // the pause, then the units
        if (at < pause) {
            u += pause - at;
            if (u >= end) break;
        }
        const int c0 = max(at - pause, 0), c1 = min(chunks, c0 + (int)(end - u));
        W.head = head;
        W.table = uni(L.a.table + (size_t)s * L.a.ldt);
        AttnRaw<G> raw;
        W.ask(rb);
        // the wave's 32 keys of each step, up to the segment's end
        const int stop = min(W.q.len, (W.q.lo & ~15) + c1 * L.unit);
        int key = (W.q.lo & ~15) + wave * 32 + c0 * L.unit;
        const int key_first = key;
        int pg[2] = {W.entry(key), W.entry(key + 16)};
        int pn[2] = {W.entry(key + AT_STEP), W.entry(key + AT_STEP + 16)};             // the table's entries, a step ahead of its loads
        if (key < stop) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint8_t *p = W.record(key + 16 * h, pg[h]);
                W.load_k(raw, h, p);
                W.load_v(raw, h, p);
            }
        }
        W.begin(rb);
#pragma clang loop unroll(disable)
        for (; key < stop; key += AT_STEP) {             // the next step's keys are on their way while one's are worked on
            const uint8_t *next[2] = {nullptr, nullptr};
            if (key + AT_STEP < stop) {
                next[0] = W.record(key + AT_STEP, pn[0]);
                next[1] = W.record(key + AT_STEP + 16, pn[1]);
            }
            const int p2[2] = {W.entry(key + 2 * AT_STEP), W.entry(key + 2 * AT_STEP + 16)};
            W.step(raw, key, pg, next);
#pragma unroll
            for (int h = 0; h < 2; h++) { pg[h] = pn[h]; pn[h] = p2[h]; }
        }
        if (__any(W.nan))
            for (int k = key_first; k < key; k += AT_STEP) at_nan<G, NT>(L, W.q, head, W.table, k, lane, W.lo, W.hi, W.o);
        const int rows = min(RB, W.q.n * L.g - rb * RB);
        auto put = [&](int r, int d, kv_f4 v) {          // 4 values of a row into out, over the row's sum of weights
            const int i = (rb * RB + r) / L.g, h = (rb * RB + r) - i * L.g;
            v *= attn_factor(sh.M[r], sh.sum[r], L.a.sink != nullptr, L.a.sink ? L.a.sink[head * L.g + h] * 1.44269504088896340736f : 0.0f);
            kv_store4(L.a.out, L.a.type, (long)(W.q.begin + i) * L.a.ldo + (long)(head * L.g + h) * L.a.hdo + d, v);
        };
        // the four waves' sums
        __syncthreads();                                 // the segment before this one has read them
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const float sum = at_sum4(W.l[t]);
            if (W.b == 0) { sh.m[wave][16 * t + W.col] = W.m[t]; sh.l[wave][16 * t + W.col] = sum; }
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int r = 16 * t + W.col;
            const float M = fmaxf(fmaxf(sh.m[0][r], sh.m[1][r]), fmaxf(sh.m[2][r], sh.m[3][r]));
            const float f = W.m[t] == -INFINITY ? 0.0f : at_exp2(W.m[t] - M);          // (a wave without keys has sums of 0 or NaN)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float *to = &sh.o[wave][r][2 * G * (4 * W.b + i)];
#pragma unroll
                for (int j = 0; j < 2 * G; j++) to[j] = W.o[t][j][i] * f;
            }
        }
        if (tid < RB) {
            float M = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++) M = fmaxf(M, sh.m[k][tid]);
#pragma unroll
            for (int k = 0; k < 4; k++) sum += sh.l[k][tid] * (sh.m[k][tid] == -INFINITY ? 0.0f : at_exp2(sh.m[k][tid] - M));
            sh.M[tid] = M;
            sh.sum[tid] = sum;
        }
        __syncthreads();
        const bool whole = c0 == 0 && c1 == chunks;
        // Pieces go through accesses of device scope (sc1), which no XCD's L2 holds back or stale: no cache is written back or
        // emptied (a fence of that scope in each of some hundred workgroups took 200 us).
        auto piece = [&](uint32_t k, uint32_t first) { return (2 * k + (k == first)) * (uint32_t)(PIECE * 4); };
        auto get4 = [&](uint32_t at) { return __builtin_bit_cast(kv_f4, __builtin_amdgcn_raw_buffer_load_b128(pieces, at, 0, AT_SC1)); };
        auto get = [&](uint32_t at) { return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(pieces, at, 0, AT_SC1)); };
        auto set4 = [&](uint32_t at, kv_f4 v) { __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(at_u4, v), pieces, at, 0, AT_SC1); };
        auto set = [&](uint32_t at, float v) { __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), pieces, at, 0, AT_SC1); };
        const uint32_t wA = whole ? w : runs.owner(u - c0), wB = whole ? w : runs.owner(u - c0 + chunks - 1);
        const uint32_t mine_at = piece(w, wA);
        for (int x = tid; x < rows * (D / 4); x += 256) {
            const int r = x / (D / 4), d = x % (D / 4) * 4;
            kv_f4 v = *(const kv_f4 *)&sh.o[0][r][d];
#pragma unroll
            for (int k = 1; k < 4; k++) v += *(const kv_f4 *)&sh.o[k][r][d];
            if (whole) put(r, d, v);
            else set4(mine_at + (r * D + d) * 4, v);
        }
        if (!whole) {
            if (tid < rows) {
                set(mine_at + (RB * D + tid) * 4, sh.M[tid]);
                set(mine_at + (RB * D + RB + tid) * 4, sh.sum[tid]);
            }
            // Pieces wA .. wB are joined in groups of `size`, then the groups' sums: whoever comes last joins.
            const uint32_t n = wB - wA + 1;
            uint32_t size = n;
            // (32 pieces of 4 rows of 128 values are faster joined at once, of 16 rows of 256 in two levels: 37 us and 31 in all)
            if (n > AT_JOIN || n * (uint32_t)(rows * D) > 1u << 16) size = (uint32_t)ceilf(sqrtf((float)n));      // 23 of 512
            const uint32_t groups = (n + size - 1) / size;
            auto last = [&](int *count, uint32_t of) {   // whether the others have all written theirs
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                       // they are in memory
                __syncthreads();
                if (tid == 0) {
                    sh.last = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == (int)of;
                    if (sh.last) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                __syncthreads();
                return sh.last != 0;
            };
            // Pieces first, first + step, .. (count of them, AT_JOIN at most) into out, or into the first of them.  `split`
            // neighbouring lanes share 4 values of a row, and load their pieces 16 at a time, the first before the factors are known.
            auto join = [&](uint32_t first, uint32_t step, int count, bool end_) {
                const int n4 = rows * (D / 4), lg = n4 <= 32 ? 3 : n4 <= 64 ? 2 : n4 <= 128 ? 1 : 0, split = 1 << lg, sub = tid & (split - 1);
                auto from = [&](int k) { return piece(first + k * step, wA); };
                kv_f4 y[16];
                auto load = [&](int x, int k0) {
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        const int at = k0 + k * split + sub;
                        if (k0 + k * split < count) y[k] = get4(from(min(at, count - 1)) + min(x, n4 - 1) * 16);
                    }
                };
                load(tid >> lg, 0);
                for (int x = tid; x < count * rows; x += 256) {
                    const int k = x / rows, r = x - k * rows;
                    sh.j.m[k][r] = get(from(k) + (RB * D + r) * 4);
                    sh.j.l[k][r] = get(from(k) + (RB * D + RB + r) * 4);
                }
                __syncthreads();
                if (tid < rows) {
                    float M = -INFINITY, sum = 0.0f;
                    for (int k = 0; k < count; k++) M = fmaxf(M, sh.j.m[k][tid]);
                    for (int k = 0; k < count; k++) {
                        const float f = sh.j.m[k][tid] == -INFINITY ? 0.0f : at_exp2(sh.j.m[k][tid] - M);
                        sum += sh.j.l[k][tid] * f;
                        sh.j.m[k][tid] = f;
                    }
                    sh.M[tid] = M;
                    sh.sum[tid] = sum;
                }
                __syncthreads();
                for (int x = tid >> lg; x < n4; x += 256 >> lg) {
                    const int r = x / (D / 4), d = x % (D / 4) * 4;
                    kv_f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
                    for (int k0 = 0; k0 < count; k0 += 16 * split) {
                        if (k0 > 0 || x != tid >> lg) load(x, k0);
#pragma unroll
                        for (int k = 0; k < 16; k++)
                            if (k0 + k * split + sub < count) v += y[k] * sh.j.m[k0 + k * split + sub][r];
                    }
                    for (int i = 1; i < split; i <<= 1) {
#pragma unroll
                        for (int e = 0; e < 4; e++) v[e] += __shfl_xor(v[e], i);
                    }
                    if (sub == 0) {
                        if (end_) put(r, d, v);
                        else set4(from(0) + x * 16, v);
                    }
                }
                if (!end_ && tid < rows) {
                    set(from(0) + (RB * D + tid) * 4, sh.M[tid]);
                    set(from(0) + (RB * D + RB + tid) * 4, sh.sum[tid]);
                }
            };
            const uint32_t group = (w - wA) / size, at = wA + group * size;
            const uint32_t in = min(size, wB + 1 - at);
            if (last(L.sync + 3 * at + (at == wA), in)) {    // (an item may end where the next begins)
                if (in > 1 || groups == 1) join(at, 1, (int)in, groups == 1);
                if (groups > 1 && last(L.sync + 3 * wA + 2, groups)) join(wA, size, (int)groups, true);
            }
        }
        u += c1 - c0;
    }
}

// ================================================================================== host side
template <int G, int NT, int PARTS>
static void attn_go(bgl_ctx *c, const AttnLaunch &L, unsigned wgs) {
    hipLaunchKernelGGL((k_attn<G, NT, PARTS>), dim3(wgs), dim3(256), 0, c->stream, L);
}
template <int G>
static void attn_pick(bgl_ctx *c, const AttnLaunch &L, int nt, unsigned wgs) {
    if constexpr (G <= 4) {
        if (nt == 2) {
            if (L.a.type == BGL_T_F32) attn_go<G, 2, 2>(c, L, wgs);
            else attn_go<G, 2, 1>(c, L, wgs);
            return;
        }
    }
    if (L.a.type == BGL_T_F32) attn_go<G, 1, 2>(c, L, wgs);
    else attn_go<G, 1, 1>(c, L, wgs);
}

// The scratch of k_attn, whose size is fixed.  A call that does without it (`needed` false) reserves it all the same, outside a capture: after any
// eager call one of single rows can be captured.
static int attn_scratch(bgl_ctx *c, bool needed) {
    const size_t part = (size_t)2 * AT_WG * 32 * (128 + 2) * 4, sync = 3 * AT_WG * sizeof(int);
    if (c->attn_part.bytes >= part && c->attn_sync.bytes >= sync) return 0;
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    if (!needed) HIPCHK(hipStreamIsCapturing(c->stream, &cs));
    if (cs != hipStreamCaptureStatusNone) return 0;
    if (const int rc = dbuf_reserve(c, c->attn_part, part, false)) return rc;
    return dbuf_reserve(c, c->attn_sync, sync, true);
}

extern "C" int bgl_attn_dev(bgl_ctx *c, const bgl_kv *kv, const bgl_attn *a) {
    if (!c || !a || !a->q || !a->out || !a->start || !a->len || !a->table) return bgl_fail(BGL_E_ARG, "bgl_attn_dev: NULL argument");
    if (const int rc = kv_check("bgl_attn_dev", kv)) return rc;
    if (a->S < 1 || a->T < 1 || a->ldt < 1) return bgl_fail(BGL_E_ARG, "bgl_attn_dev: S=%d T=%d ldt=%d", a->S, a->T, a->ldt);
    if (a->nq < 1 || a->nq > 65535 || a->nq % kv->heads)
        return bgl_fail(BGL_E_ARG, "bgl_attn_dev: nq=%d heads over a cache of %d", a->nq, kv->heads);
    if (a->type != BGL_T_F32 && a->type != BGL_T_F16 && a->type != BGL_T_BF16) return bgl_fail(BGL_E_ARG, "bgl_attn_dev: unknown element type");
    if (!kv_rows_ok(a->ldq, a->hdq, a->T, a->nq, kv->D) || !kv_rows_ok(a->ldo, a->hdo, a->T, a->nq, kv->D))
        return bgl_fail(BGL_E_ARG, "bgl_attn_dev: rows of D=%d values overlap at these strides", kv->D);
    if (a->window < 0 || (a->window && !a->causal)) return bgl_fail(BGL_E_ARG, "bgl_attn_dev: window=%d (at least 0, and with causal)", a->window);
    if (a->max_rows < 0 || a->max_len < 0) return bgl_fail(BGL_E_ARG, "bgl_attn_dev: max_rows=%d max_len=%d", a->max_rows, a->max_len);
    if (!(a->scale == a->scale) || a->scale - a->scale != 0.0f) return bgl_fail(BGL_E_ARG, "bgl_attn_dev: scale is not finite");
    if (a->q == a->out) return bgl_fail(BGL_E_ARG, "bgl_attn_dev: out is q");
    if ((long)a->T * (a->nq / kv->heads) > INT32_MAX / 2) return bgl_fail(BGL_E_ARG, "bgl_attn_dev: T=%d rows of %d heads", a->T, a->nq);
    // keys are numbered in 32 bits
    if ((long)a->ldt * kv->page > 1l << 30) return bgl_fail(BGL_E_ARG, "bgl_attn_dev: %d pages of %d tokens a sequence", a->ldt, kv->page);
    const int g = a->nq / kv->heads;
    int rows = (int)std::min<long>((long)std::min(std::max(1, a->max_rows), a->T) * g, INT32_MAX);
    // Many rows of a head at once are the prompt kernel's, where they are told of; its offsets inside a head's part of a page have 32 bits.
    const bool prompt = rows > AT_FEW && (size_t)(kv->page / KV_TILE) * kv_record(kv->D) <= 1ull << 32;
    if (prompt && ((double)a->T * g / 128 + a->S) * kv->heads > 1 << 22)        // a launch has less than 2^32 threads
        return bgl_fail(BGL_E_ARG, "bgl_attn_dev: prompts of T=%d rows of %d heads", a->T, a->nq);
    AttnLaunch L;
    memset(&L, 0, sizeof L);
    L.c = *kv;
    L.a = *a;
    L.g = g;
    L.ppt = kv->page / KV_TILE;
    L.page_bytes = (size_t)kv->heads * L.ppt * kv_record(kv->D);
    while ((1 << L.div_shift) < L.ppt) L.div_shift++;
    L.div_mul = (uint32_t)((((uint64_t)1 << 32) * ((1u << L.div_shift) - (uint32_t)L.ppt)) / L.ppt + 1);
    L.scale2 = fabsf(a->scale) * 1.44269504088896340736f;
    L.limit = INT32_MAX;
    const int G = kv->D / 32;
    // Beside prompts sequences of few rows stay here, unless it costs less to take them along as blocks that are nearly empty.
    const bool alone = prompt && attn_prompt_alone(L);
    // k_attn counts its units in 32 bits: of all rows, or beside prompts of AT_FEW for each sequence
    const double blocks = std::min((double)a->T * g / 16 + a->S, prompt ? a->S * (AT_FEW / 16.0) : INFINITY);
    if (!alone && kv->heads * blocks * ((double)a->ldt * kv->page / AT_STEP + 2 + AT_PAUSE) > 2e9)
        return bgl_fail(BGL_E_ARG, "bgl_attn_dev: T=%d rows of S=%d sequences over %d pages of %d tokens", a->T, a->S, a->ldt, kv->page);
    HIPCHK(hipSetDevice(c->device));
    // k_attn's scratch is there before the first launch: a call that fails has launched nothing.
    if (const int rc = attn_scratch(c, !alone)) return rc;
    if (prompt) {
        L.limit = alone ? 0 : AT_FEW;
        const int tok = prof_begin(c, 1);
        const int rc = run_attn_prompt(c, L);
        prof_end(c, tok);
        if (rc) return rc;
        HIPCHK(hipGetLastError());
        if (alone) return 0;
        rows = AT_FEW;
    }
    const int nt = rows > 16 && G <= 4 ? 2 : 1, RB = 16 * nt;
    L.part = (float *)c->attn_part.p;                    // (a prompt whose keys are split may have had it grow)
    L.sync = (int *)c->attn_sync.p;
    // Up to four steps stay together: a head whose keys are one unit needs no join (8 heads over 512 keys: 10.4 us in units of 128).
    const long keys = a->window ? std::min((long)a->max_len, (long)a->window + rows) : a->max_len;
    L.unit = keys <= 4 * AT_STEP ? 4 * AT_STEP : AT_STEP;
    const long chunks = (std::max(1l, keys) + L.unit - 1) / L.unit, units = (long)a->S * kv->heads * ((rows + RB - 1) / RB) * chunks;
    // Two units for a workgroup, where an item's pieces are large or many: half of them to join (2 sequences of 4096 keys, 2 heads of 128, 16 rows:
    // 19.4 us in 128 workgroups, 15.8 in 64; 8 heads of 128, 4 rows: 8192 keys 15.2 and 13.7, 3000 keys 11.6 and 12.1).
    L.least = chunks * std::min(rows, RB) * kv->D > 1 << 14 ? 2 : 1;
    const unsigned wgs = (unsigned)std::min<long>(AT_WG, std::max<long>(1, units < 128 ? units : units / L.least));
    const int tok = prof_begin(c, 1);
    switch (G) {
    case 2: attn_pick<2>(c, L, nt, wgs); break;
    case 3: attn_pick<3>(c, L, nt, wgs); break;
    case 4: attn_pick<4>(c, L, nt, wgs); break;
    case 6: attn_pick<6>(c, L, nt, wgs); break;
    default: attn_pick<8>(c, L, nt, wgs); break;
    }
    prof_end(c, tok);
    HIPCHK(hipGetLastError());
    return 0;
}
