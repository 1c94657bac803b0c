// bgl_moe_i8.hip -- a routed FFN (moe_ffn_batched, qwen_infer.c:5238-5350) of K_Q8C experts for a few tokens:
//
//   xq, xs = the int8 codes of each token
//   g, u   = gate_e xq, up_e xq ; h = silu(g) * u   per pair (token, expert); the shared experts: per token
//   hq, hs = the int8 codes of each h row
//   out[t] = sum_e w_e * down_e hq (ascending expert ids) + shared down
//
// with the products of bgl_i8.hip (exact int32 sums, then fp32 operations in the order written there), so a
// row's bits depend neither on the other tokens nor on how the work is split.
//
// What bounds it is the experts' bytes: each touched expert is read once for up to 16 of its tokens (64 tokens
// at the most; more go in chunks).  All of it is one launch, k_moe_i8, whose workgroups have four roles:
//   i8_pre           codes of x; the router's scores, a wave an expert, and the softmax and top-K of a token by
//                    its last workgroup
//   i8_gate_up       16-row blocks of both tensors, the shared experts' while the routing is made, then the used experts'
//                    in equal runs, whose waves split K; the next block's operands are on their way while one is
//                    multiplied.  Whoever finishes an expert's last block makes the codes of its h rows.
//   i8_shared_codes  codes of the shared experts' h
//   i8_down          a workgroup owns 8 output channels; its waves take pieces of the experts' K, the first two of which
//                    they load before they wait for h, and add the int32 sums in LDS, which holds every pair's until the
//                    combine: no memory traffic for partial sums
// Workgroups wait only for ones with lower ids, and find their expert and its pairs from the routing themselves.  1024
// threads with up to 128 registers fill a CU, so that equal shares take equal times (with 512 threads a CU often had two
// workgroups of down and its neighbour none: 173 us for 32 tokens, and 161 as four launches).
// 64 experts of 2048 x 1408, 6 a token, a shared 2816, three layers' weights and seven sets of tokens in turn in a graph:
// 1 token 31 us (four launches 41), 8 tokens 77 (96), 32 tokens 130 (161), 64 tokens 155 (204), 128 as two launches 309.
// (With the same token's experts in the last-level cache 1 token takes 28.6.)  32 tokens' gate and up move 4.9 TB/s, a large copy 5.1; what is above the bytes' time is the
// routing (9 us at one token from the first load to the last workgroup's list, of which 2.4 the top-K), the codes between
// the last h and down's products (6) and the slowest CU's share.
#include <string.h>

#include <algorithm>

#include "../../include/beglin_qgemv.h"
#include "bgl_i8.h"
#include "bgl_route.h"

#define HIPCHK(expr)                                                                             \
    do {                                                                                         \
        hipError_t e_ = (expr);                                                                  \
        if (e_ != hipSuccess) return bgl_fail(BGL_E_HIP, "%s: %s", #expr, hipGetErrorString(e_)); \
    } while (0)

#define MOE_I8_TOK 64             // tokens of a chunk
#define MOE_I8_PAIRS (MOE_I8_TOK * MOE_MAX_K)
#define MOE_I8_NT 1024            // threads of a workgroup: one a CU, so that equal shares take equal times
#define MOE_I8_NW (MOE_I8_NT / 64)
#define MOE_I8_FEW 32             // pairs whose routing one wave does (1 token of 6 34.6 -> 33.7 us; at 48 pairs 82 -> 85)
#define MOE_I8_DC 6               // units of 128 values that a down wave takes at a time at most (8: 132 us for 129 at 32 tokens)
#define MOE_I8_GU_WGS 256         // gate+up workgroups at most
#define MOE_I8_SQ 4               // tokens whose shared h one workgroup makes the codes of
#define MOE_I8_SQ_WGS (MOE_I8_TOK / MOE_I8_SQ)
#define MOE_I8_WGS (MOE_I8_TOK + MOE_I8_TOK * ROUTE_MAXE / MOE_I8_NW + MOE_I8_GU_WGS + MOE_I8_SQ_WGS + 131072 / 8)   // of a launch

// What the workgroups of a launch tell each other.  Each flag holds the number of the last launch that set it.
struct MoeI8Sync {
    int gave_up, pad[15];                // a wait ended at its limit (bgl_ctx_check)
    int codes[MOE_I8_TOK];               // a token's codes are there
    int shared[MOE_I8_GU_WGS];           // a gate+up workgroup's share of the shared experts is done
    int gu[MOE_I8_GU_WGS];               // all it does
    int sq[MOE_I8_SQ_WGS];               // codes of the shared experts' h are there
    // 16-row blocks of a slot that are done, in the half of the launch's number; each launch zeroes the next one's half, so
    // that counts which waits that gave up left wrong are nobody's
    int blocks[2][MOE_I8_PAIRS];
    int gen[MOE_I8_WGS];                 // launches so far: the same in every element between launches
    // values that carry the number of their launch in the upper half
    uint64_t score[MOE_I8_TOK * ROUTE_MAXE], idx[MOE_I8_PAIRS], w[MOE_I8_PAIRS];
};

struct MoeI8Launch {
    const BglDevTensor *tg, *tu, *td;    // expert tables
    BglDevTensor sg, su, sd;             // shared experts (shared != 0)
    int shared, E, K, T, P, H, I, Ish, nslots, piece;   // nslots: the most slots; piece: units a down wave takes
    int hp, ip, ishp;                    // bytes of a row of codes: a multiple of 128, so that no two share a line
    int npre, ngu, nsq;                  // workgroups of each role; the rest is down's
    int never, spin;                     // a test's launch, in whose odd workgroups waits give up; polls before a wait does
    MoeI8Sync *sync;
    const float *x, *rw, *rb;            // token rows; router
    int renorm;
    const int32_t *idx;                  // [P] and their weights, or null: the router's, in sync
    const float *w;
    int8_t *xq;
    float *xs;
    float *h, *hsh;                      // [P][I], [T][Ish]
    int8_t *hq, *hshq;                   // codes of h and their scales [P + T]
    float *hs;
    float *out;
};

// What one workgroup writes and another reads in the same launch passes the L2s of the eight dies: stores at agent scope,
// and loads at agent scope too wherever the line could be in the reader's L2 before.
template <class T> __device__ __forceinline__ void i8_put(T *p, T v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <class T> __device__ __forceinline__ T i8_get(const T *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ i8_f4 i8_get4(const float *p) {
    const uint64_t a = i8_get((const uint64_t *)p), b = i8_get((const uint64_t *)p + 1);
    return i8_f4{__uint_as_float((uint32_t)a), __uint_as_float((uint32_t)(a >> 32)), __uint_as_float((uint32_t)b), __uint_as_float((uint32_t)(b >> 32))};
}
// what a wait waits for
__device__ __forceinline__ int i8_expect(const MoeI8Launch &L, int gen) { return gen + (L.never & (int)blockIdx.x); }
// A value and the number of its launch in one store; and the wait for it, by one lane.
__device__ __forceinline__ void i8_put_now(uint64_t *p, int gen, uint32_t v) { i8_put(p, (uint64_t)(uint32_t)gen << 32 | v); }
__device__ __forceinline__ uint32_t i8_get_now(const MoeI8Launch &L, const uint64_t *p, int gen) {
    for (int s = 0;;) {
        const uint64_t v = i8_get(p);
        if ((int)(v >> 32) == i8_expect(L, gen)) return (uint32_t)v;
        if (++s >= L.spin) break;
        __builtin_amdgcn_s_sleep(1);
    }
    i8_put(&L.sync->gave_up, 1);
    return 0xffffffffu;
}
__device__ __forceinline__ int i8_idx(const MoeI8Launch &L, int p, int gen) { return L.idx ? L.idx[p] : (int)i8_get_now(L, L.sync->idx + p, gen); }
__device__ __forceinline__ float i8_weight(const MoeI8Launch &L, int p, int gen) { return L.w ? L.w[p] : __uint_as_float(i8_get_now(L, L.sync->w + p, gen)); }
// the workgroup's stores are in memory, and then its flag
__device__ __forceinline__ void i8_done(int *flag, int gen) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) i8_put(flag, gen);
}
// Waits until n flags show `gen`; all threads call it.  A workgroup waits for ones with lower ids only, which are
// dispatched before it and wait for none behind them; after `spin` polls it goes on with what is there.
__device__ __forceinline__ void i8_wait(const MoeI8Launch &L, const int *flag, int n, int gen) {
    if (threadIdx.x < 64) {
        for (int s = 0;;) {
            bool ok = true;
            for (int i = threadIdx.x; i < n; i += 256) {       // four loads at a time
                int v[4];
#pragma unroll
                for (int j = 0; j < 4; j++) v[j] = i8_get(flag + min(i + 64 * j, n - 1));
#pragma unroll
                for (int j = 0; j < 4; j++) ok &= v[j] == i8_expect(L, gen);
            }
            if (__builtin_amdgcn_ballot_w64(!ok) == 0) break;
            if (++s >= L.spin) {
                if (threadIdx.x == 0) i8_put(&L.sync->gave_up, 1);
                break;
            }
            __builtin_amdgcn_s_sleep(1);
        }
    }
    __syncthreads();
}

// ------------------------------------------------------------------ codes of rows, routing
// The codes and scales of n rows by the workgroup; row(i) is row i's number in all of the arrays, and COH: they were written
// in this launch.  16 lanes take 64 values, which belong to one row.  Up to 16384 values stay in registers between the
// maxima and the codes.  mx: an LDS word a row.
template <bool COH, class Row>
__device__ __forceinline__ void i8_row_codes(const float *x, int width, int8_t *q, int pitch, float *scale, int n, uint32_t *mx, Row row) {
    constexpr int RND = 4, GRP = MOE_I8_NT / 16;
    const int tid = threadIdx.x, per = width / 64, nch = n * per;
    i8_f4 v[RND];
    auto load = [&](int c0) {
#pragma unroll
        for (int r = 0; r < RND; r++) {
            if (c0 + r * GRP >= nch) break;
            const int ch = min(c0 + r * GRP + (tid >> 4), nch - 1), i = ch / per;
            const float *p = x + (size_t)row(i) * width + (ch - i * per) * 64 + 4 * (tid & 15);
            v[r] = COH ? i8_get4(p) : i8_f4{p[0], p[1], p[2], p[3]};
        }
    };
    __syncthreads();                                           // (LDS may hold an earlier role's or slot's)
    for (int i = tid; i < n; i += MOE_I8_NT) mx[i] = I8_MX0;
    __syncthreads();
    for (int c0 = 0; c0 < nch; c0 += RND * GRP) {
        load(c0);
#pragma unroll
        for (int r = 0; r < RND; r++) {
            if (c0 + r * GRP >= nch) break;
            uint32_t mb = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) mb = max(mb, __float_as_uint(v[r][j]) & 0x7fffffffu);
            mb = max(mb, (uint32_t)dpp_i<0xB1>((int)mb));
            mb = max(mb, (uint32_t)dpp_i<0x4E>((int)mb));
            mb = max(mb, (uint32_t)dpp_i<0x141>((int)mb));
            mb = max(mb, (uint32_t)dpp_i<0x140>((int)mb));
            if ((tid & 15) == 0) atomicMax(&mx[min(c0 + r * GRP + (tid >> 4), nch - 1) / per], mb);
        }
    }
    __syncthreads();
    for (int c0 = 0; c0 < nch; c0 += RND * GRP) {
        if (nch > RND * GRP) load(c0);
#pragma unroll
        for (int r = 0; r < RND; r++) {
            const int ch = c0 + r * GRP + (tid >> 4), i = ch / per;
            if (ch >= nch) break;
            const I8Scale s = i8_scale(mx[i]);
            i8_put((uint32_t *)(q + (size_t)row(i) * pitch + (ch - i * per) * 64 + 4 * (tid & 15)),
                   i8_pack4(i8_code(v[r].x, s), i8_code(v[r].y, s), i8_code(v[r].z, s), i8_code(v[r].w, s)));
        }
    }
    for (int i = tid; i < n; i += MOE_I8_NT) i8_put(scale + row(i), i8_scale(mx[i]).sc);
}

// Workgroups [0, T): a token's codes.  The others: a wave an expert's score; a token's last one takes the softmax and the
// top-K when the others' scores are there.
__device__ __forceinline__ void i8_pre(const MoeI8Launch &L, int b, int gen, uint8_t *lds) {
    const int tid = threadIdx.x, lane = tid & 63;
    if (b < L.T) {
        i8_row_codes<false>(L.x, L.H, L.xq, L.hp, L.xs, 1, (uint32_t *)lds, [&](int) { return b; });
        i8_done(L.sync->codes + b, gen);
        return;
    }
    const int per = (L.E + MOE_I8_NW - 1) / MOE_I8_NW, t = (b - L.T) / per, e = ((b - L.T) % per) * MOE_I8_NW + (tid >> 6);
    float *const lbuf = (float *)lds, *const sc = lbuf + ROUTE_MAXE;
    if (e < L.E) {
        const double acc = route_dot_wave(L.rw + (size_t)e * L.H, L.x + (size_t)t * L.H, L.H, lane);
        const float s = L.rb ? __fadd_rn((float)acc, L.rb[e]) : (float)acc;
        if (lane == 0) i8_put_now(L.sync->score + t * ROUTE_MAXE + e, gen, __float_as_uint(s));
    }
    if ((b - L.T) % per != per - 1 || tid >= 64) return;
    for (int i = lane; i < L.E; i += 64) sc[i] = __uint_as_float(i8_get_now(L, L.sync->score + t * ROUTE_MAXE + i, gen));
    __builtin_amdgcn_wave_barrier();
    float sel_w;
    int sel_i;
    route_topk_wave(sc, L.E, L.K, L.renorm, lane, sel_i, sel_w, lbuf);
    if (lane < L.K && sel_i >= L.E) {                          // scores of which one is NaN or +Inf pick nothing: the sum is NaN
        sel_i = lane;
        sel_w = __uint_as_float(0x7fc00000u);
    }
    if (lane < L.K) {
        i8_put_now(L.sync->idx + t * L.K + lane, gen, (uint32_t)sel_i);
        i8_put_now(L.sync->w + t * L.K + lane, gen, __float_as_uint(sel_w));
    }
}

// ------------------------------------------------------------------ the routing in LDS
// The used experts in ascending order ("slots") and each one's pairs.  (The order of a slot's pairs is that of LDS
// atomics; no value depends on it.)
#define MOE_I8_NONE 0xffff
struct MoeI8Route {
    uint16_t slot[MOE_I8_PAIRS];         // of each pair; MOE_I8_NONE: its id lies outside the stack
    uint16_t list[MOE_I8_PAIRS];         // the pairs by slot
    uint16_t expert[MOE_I8_PAIRS];       // of each slot
    int off[MOE_I8_PAIRS + 1], at[MOE_I8_PAIRS];
    uint32_t used[32], base[32];         // experts that have a pair (E <= 1024), slots before each 32 of them
    int n;                               // slots
};
__device__ __forceinline__ void i8_routing(const MoeI8Launch &L, MoeI8Route &R, int gen) {
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 63;
    // few pairs: a lane each, without the barriers
    if (L.P <= MOE_I8_FEW) {
        if (tid < 64) {
            const int got = lane < L.P ? i8_idx(L, lane, gen) : -1, e = got >= 0 && got < L.E ? got : 0x7fffffff;
            int s = 0, less = 0, n = 0;
            uint64_t same = 0;
            for (int p = 0; p < L.P; p++) {
                const int o = __builtin_amdgcn_readlane(e, p);
                const uint64_t m = __builtin_amdgcn_ballot_w64(e == o);
                const int first = o != 0x7fffffff && __builtin_ctzll(m) == p;
                if (o < e) { s += first; less++; }
                if (o == e) same = m;
                n += first;
            }
            const int before = __popcll(same & ((1ull << lane) - 1));
            if (lane < L.P) {
                const bool ok = e != 0x7fffffff;
                R.slot[lane] = ok ? (uint16_t)s : (uint16_t)MOE_I8_NONE;
                if (ok) {
                    R.list[less + before] = (uint16_t)lane;
                    R.expert[s] = (uint16_t)e;
                    R.off[s] = less;
                    if (s == n - 1) R.off[n] = less + __popcll(same);
                }
            }
            if (lane == 0) R.n = n;
        }
        __syncthreads();
        return;
    }
    if (tid < 32) R.used[tid] = 0;
    for (int s = tid; s < L.nslots; s += nt) R.at[s] = 0;
    __syncthreads();
    for (int p = tid; p < L.P; p += nt) {
        const int e = i8_idx(L, p, gen);
        R.slot[p] = e >= 0 && e < L.E ? (uint16_t)e : (uint16_t)MOE_I8_NONE;     // the expert, for now
        if (e >= 0 && e < L.E) atomicOr(&R.used[e >> 5], 1u << (e & 31));
    }
    __syncthreads();
    if (tid < 64) {
        const int c = lane < 32 ? __popc(R.used[lane]) : 0;
        int incl = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up(incl, o);
            if (lane >= o) incl += v;
        }
        if (lane < 32) R.base[lane] = incl - c;
        if (lane == 31) R.n = incl;
    }
    __syncthreads();
    for (int p = tid; p < L.P; p += nt) {
        const uint32_t e = R.slot[p];
        if (e == MOE_I8_NONE) continue;
        const int s = R.base[e >> 5] + __popc(R.used[e >> 5] & ((1u << (e & 31)) - 1));
        R.slot[p] = (uint16_t)s;
        R.expert[s] = (uint16_t)e;
        atomicAdd(&R.at[s], 1);
    }
    __syncthreads();
    if (tid < 64) {
        int before = 0;
        for (int s0 = 0; s0 < R.n; s0 += 64) {
            const int c = s0 + lane < R.n ? R.at[s0 + lane] : 0;
            int incl = c;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int v = __shfl_up(incl, o);
                if (lane >= o) incl += v;
            }
            if (s0 + lane < R.n) R.off[s0 + lane] = R.at[s0 + lane] = before + incl - c;
            before += __shfl(incl, 63);
        }
        if (lane == 0) R.off[R.n] = before;
    }
    __syncthreads();
    for (int p = tid; p < L.P; p += nt) {
        const int s = R.slot[p];
        if (s != MOE_I8_NONE) R.list[atomicAdd(&R.at[s], 1)] = (uint16_t)p;
    }
    __syncthreads();
}

__device__ __forceinline__ i8_i4 mi_mfma(i8_u4 a, i8_u4 b, i8_i4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i8_i4, a), __builtin_bit_cast(i8_i4, b), c, 0, 0, 0);
}
// A pointer that every lane has alike, from a table: in scalar registers and known to be global memory (a load through a
// pointer that might be LDS waits for all that are out).
typedef const __attribute__((address_space(1))) uint8_t *i8_gp;
__device__ __forceinline__ i8_gp mi_uniform(const void *p) {
    const uint64_t v = (uint64_t)p;
    return (i8_gp)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v) | (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32);
}
__device__ __forceinline__ i8_u4 mi_load(i8_gp base, uint32_t off) { return *(const __attribute__((address_space(1))) i8_u4 *)(base + off); }
__device__ __forceinline__ float mi_float(i8_gp base, int i) { return ((const __attribute__((address_space(1))) float *)base)[i]; }

// ------------------------------------------------------------------ gate + up
// h of the 16-row blocks rb0 .. rb1 - 1 for the 16 columns from c0 of the n in list (a pair, or with list null a token).  A
// wave takes every 16th unit of K, two at a time, and has the operands of its next two on their way while it multiplies.  par: which of two LDS buffers holds the next sums, so that one barrier a block is enough.
#define MOE_I8_RED 148            // int32 x 4 of a wave's sums of both tensors, placed so that a wave reads 64 banks
__device__ __forceinline__ void i8_gu(const MoeI8Launch &L, const BglDevTensor &G, const BglDevTensor &Up, int rb0, int rb1, const uint16_t *list,
                                      int c0, int n, float *h, int width, i8_i4 *red, int &par) {
    constexpr int D = 2;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int U = L.H / 64, NC = (U + D * MOE_I8_NW - 1) / (D * MOE_I8_NW), its = (rb1 - rb0) * NC, cpr = (L.H + 127) / 128 * 8;
    const i8_gp gw = mi_uniform(G.w), uw = mi_uniform(Up.w), gsc = mi_uniform(G.s0), usc = mi_uniform(Up.s0), xq = (i8_gp)L.xq;
    const uint32_t lo = (lane >> 4) * 1024 + (lane & 15) * 16;   // of a lane's operand in 16 rows' unit
    const int xc = min(c0 + (lane & 15), n - 1);
    const uint32_t xo = (list ? list[xc] / L.K : xc) * L.hp + (lane >> 4) * 16;
    // a thread sums a quarter of the waves for channel och of column oc
    const int och = tid >> 2 & 15, oc = c0 + (tid >> 6), orow = list ? list[min(oc, n - 1)] : min(oc, n - 1);
    const float xs = i8_get(L.xs + (list ? orow / L.K : orow));
    struct Ops { i8_u4 x[D], a[D], b[D]; } even, odd;          // in turn: no copy waits for a load
    auto load = [&](Ops &o, int it) {
        const int rb = rb0 + it / NC, u0 = (it % NC) * D * MOE_I8_NW + wave;
        const size_t at = (size_t)(rb >> 2) * cpr * 1024 + (rb & 3) * 256;
#pragma unroll
        for (int s = 0; s < D; s++) {
            const int u = min(u0 + s * MOE_I8_NW, U - 1);
            o.x[s] = mi_load(xq + u * 64, xo);
            o.a[s] = mi_load(gw + at + (size_t)u * 4096, lo);
            o.b[s] = mi_load(uw + at + (size_t)u * 4096, lo);
        }
    };
    i8_i4 ga, ua;
    float gs = 0.0f, us = 0.0f;
    auto step = [&](int it, const Ops &cur, Ops &next) {
        const int ch = it % NC, rb = rb0 + it / NC, u0 = ch * D * MOE_I8_NW + wave;
        if (ch == 0) {
            ga = ua = i8_i4{0, 0, 0, 0};
            gs = mi_float(gsc + 64 * (size_t)rb, och);
            us = mi_float(usc + 64 * (size_t)rb, och);
        }
        load(next, min(it + 1, its - 1));
#pragma unroll
        for (int s = 0; s < D; s++)
            if (u0 + s * MOE_I8_NW < U) {
                ga = mi_mfma(cur.a[s], cur.x[s], ga);
                ua = mi_mfma(cur.b[s], cur.x[s], ua);
            }
        if (ch != NC - 1) return;
        i8_i4 *const r = red + par * MOE_I8_NW * MOE_I8_RED;
        r[wave * MOE_I8_RED + lane + (lane >> 4)] = ga;
        r[wave * MOE_I8_RED + lane + (lane >> 4) + 68] = ua;
        __syncthreads();
        par ^= 1;
        const int *s = (const int *)r + ((och >> 2) * 17 + (tid >> 6)) * 4 + (och & 3);
        int g = 0, u = 0;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const int *v = s + ((tid & 3) + 4 * w) * MOE_I8_RED * 4;
            g += v[0];
            u += v[68 * 4];
        }
        g += dpp_i<0xB1>(g); u += dpp_i<0xB1>(u);
        g += dpp_i<0x4E>(g); u += dpp_i<0x4E>(u);
        if ((tid & 3) == 0 && oc < n) i8_put(h + (size_t)orow * width + 16 * rb + och, i8_swiglu(i8_out(g, xs, gs), i8_out(u, xs, us)));
    };
    load(even, 0);
    for (int it = 0; it < its; it += 2) {
        step(it, even, odd);
        if (it + 1 < its) step(it + 1, odd, even);
    }
}

// The 16-row blocks of the shared experts, which wait for the codes only, and then those of the used experts, each in equal
// runs over the workgroups.  Whoever finds that a slot's last block is done makes the codes of its rows.
__device__ __forceinline__ void i8_gate_up(const MoeI8Launch &L, int b, int gen, MoeI8Route &R, uint8_t *lds) {
    i8_i4 *const red = (i8_i4 *)lds;                           // [2][wave][MOE_I8_RED]
    int par = 0;
    i8_wait(L, L.sync->codes, L.T, gen);
    if (L.shared) {
        // (not over the last ones, which start when the scores' workgroups leave their CUs)
        const int nsh = L.Ish / 16, ns = L.ngu - min(L.npre, L.ngu / 4);
        const int rb0 = (int)((long)nsh * min(b, ns) / ns), rb1 = (int)((long)nsh * min(b + 1, ns) / ns);
        if (rb0 < rb1)
            for (int c0 = 0; c0 < L.T; c0 += 16) i8_gu(L, L.sg, L.su, rb0, rb1, nullptr, c0, L.T, L.hsh, L.Ish, red, par);
        i8_done(L.sync->shared + b, gen);
    }
    i8_routing(L, R, gen);
    const int per = L.I / 16;
    const long all = (long)__builtin_amdgcn_readfirstlane(R.n) * per;
    const int begin = (int)(all * b / L.ngu), end = (int)(all * (b + 1) / L.ngu);
    for (int it = begin; it < end;) {
        const int slot = it / per, first = slot * per, rb1 = min(end - first, per);
        const int e = __builtin_amdgcn_readfirstlane((int)R.expert[slot]);
        const int l0 = __builtin_amdgcn_readfirstlane(R.off[slot]), n = __builtin_amdgcn_readfirstlane(R.off[slot + 1]) - l0;
        const BglDevTensor G = L.tg[e], U = L.tu[e];
        for (int c0 = 0; c0 < n; c0 += 16) i8_gu(L, G, U, it - first, rb1, R.list + l0, c0, n, L.h, L.I, red, par);
        it = first + rb1;
    }
    // (a run has less than 64 slots: at most 1024 of them over 256 workgroups)
    uint64_t *const whole = (uint64_t *)lds;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");           // h is in memory before the blocks are counted
    __syncthreads();
    if (threadIdx.x < 64) {
        const int s = begin / per + (int)threadIdx.x, n = min(end, (s + 1) * per) - max(begin, s * per);
        bool last = false;
        if (n > 0 && begin < end)
            last = __hip_atomic_fetch_add(L.sync->blocks[gen & 1] + s, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + n == per;
        const uint64_t m = __builtin_amdgcn_ballot_w64(last);
        if (threadIdx.x == 0) *whole = m;
    }
    __syncthreads();
    for (uint64_t m = *whole; m; m &= m - 1) {                 // (uniform)
        const int s = begin / per + __builtin_ctzll(m);
        const uint16_t *const list = R.list + R.off[s];
        i8_row_codes<true>(L.h, L.I, L.hq, L.ip, L.hs, R.off[s + 1] - R.off[s], (uint32_t *)lds + 2, [&](int i) { return (int)list[i]; });
    }
    i8_done(L.sync->gu + b, gen);
}

// ------------------------------------------------------------------ codes of the shared experts' h
__device__ __forceinline__ void i8_shared_codes(const MoeI8Launch &L, int b, int gen, uint8_t *lds) {
    i8_wait(L, L.sync->shared, L.ngu, gen);
    const int t0 = b * MOE_I8_SQ;
    i8_row_codes<true>(L.hsh, L.Ish, L.hshq, L.ishp, L.hs + L.P, min(L.T - t0, MOE_I8_SQ), (uint32_t *)lds, [&](int i) { return t0 + i; });
    i8_done(L.sync->sq + b, gen);
}

// ------------------------------------------------------------------ down + combine
// A workgroup owns 8 output channels rb.  An operand of 16 rows is these channels twice, for 64 values of K and the next
// 64, against 8 columns twice, so that all CUs have a workgroup; the quarters of the product where the two belong together
// are used.
struct MoeI8Down {                       // dynamic LDS of a down workgroup
    int sums, tw, ts, order;
    __device__ MoeI8Down(const MoeI8Launch &L) {
        const int rows = L.P + (L.shared ? L.T : 0);
        sums = 0;                        // int [P + T][8]
        tw = rows * 32;                  // each slot's weights and scales
        ts = tw + L.nslots * 8;
        order = ts + L.nslots * 8;       // uint16 [P]
    }
};
__device__ __forceinline__ void i8_down(const MoeI8Launch &L, int rb, int gen, MoeI8Route &R, uint8_t *lds) {
    const MoeI8Down at(L);
    int *const sums = (int *)(lds + at.sums);
    const uint8_t **const tw = (const uint8_t **)(lds + at.tw);
    const float **const ts = (const float **)(lds + at.ts);
    uint16_t *const order = (uint16_t *)(lds + at.order);
    const int rows = L.P + (L.shared ? L.T : 0), tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    for (int i = tid; i < rows * 8; i += MOE_I8_NT) sums[i] = 0;
    i8_routing(L, R, gen);
    const int nslots = __builtin_amdgcn_readfirstlane(R.n);
    for (int s = tid; s < nslots; s += MOE_I8_NT) {
        tw[s] = L.td[R.expert[s]].w;
        ts[s] = (const float *)L.td[R.expert[s]].s0;
    }
    __syncthreads();
    // pieces of the shared experts first (the longest rows), then of the routed ones
    const int U = (L.I + 127) / 128, Us = (L.Ish + 127) / 128;
    const int np = (U + L.piece - 1) / L.piece, nps = L.shared ? (Us + L.piece - 1) / L.piece : 0, tasks = nps + nslots * np;
    const size_t lw = (size_t)(rb >> 3) * 8192;
    const uint32_t lo = (lane >> 3 & 1) * 4096 + (lane >> 4) * 1024 + ((rb & 7) * 8 + (lane & 7)) * 16;
    struct Piece { int slot, u0, nu; i8_u4 a[MOE_I8_DC]; } even, odd;      // in turn: no copy waits for a load
    // a piece's place and weights
    auto fetch = [&](Piece &p, int task) {
        const bool sh = task < nps;
        p.slot = sh ? -1 : (task - nps) / np;
        p.u0 = (sh ? task : (task - nps) % np) * L.piece;
        p.nu = min(L.piece, (sh ? Us : U) - p.u0);
        const i8_gp wp = mi_uniform(sh ? L.sd.w : tw[p.slot]) + lw * (sh ? Us : U) + (size_t)p.u0 * 8192;
#pragma unroll
        for (int s = 0; s < MOE_I8_DC; s++) p.a[s] = mi_load(wp + (size_t)min(s, p.nu - 1) * 8192, lo);
    };
    // on their way while gate+up ends
    if (wave < tasks) fetch(even, wave);
    if (wave + MOE_I8_NW < tasks) fetch(odd, wave + MOE_I8_NW);
    // a token's pairs by expert, then k: the order in which they are added
    for (int p = tid; p < L.P; p += MOE_I8_NT) {
        const int t = p / L.K, me = R.slot[p];
        int before = 0;
        for (int o = t * L.K; o < (t + 1) * L.K; o++) before += R.slot[o] < me || (R.slot[o] == me && o < p);
        order[t * L.K + before] = (uint16_t)p;
    }
    i8_wait(L, L.sync->gu, L.ngu, gen);
    if (L.shared) i8_wait(L, L.sync->sq, L.nsq, gen);
    const bool used = (lane >> 3 & 1) == lane >> 5;              // (channel 4 * (lane >> 4 & 1) + i, column lane & 7)
    auto piece = [&](int task, const Piece &cur, Piece &nxt) {
        const bool sh = cur.slot < 0;
        const int l0 = sh ? 0 : R.off[cur.slot], n = sh ? L.T : R.off[cur.slot + 1] - l0;
        const i8_gp codes = (i8_gp)(sh ? L.hshq : L.hq) + cur.u0 * 128;
        for (int c0 = 0; c0 < n; c0 += 8) {
            const int c = min(c0 + (lane & 7), n - 1), row = sh ? c : R.list[l0 + c];
            const uint32_t xo = row * (sh ? L.ishp : L.ip) + (lane >> 3 & 1) * 64 + (lane >> 4) * 16;
            i8_i4 acc = {0, 0, 0, 0};
            i8_u4 x[MOE_I8_DC];
#pragma unroll
            for (int s = 0; s < MOE_I8_DC; s++) x[s] = mi_load(codes + min(s, cur.nu - 1) * 128, xo);
            // behind the codes: loads return in order, and these are waited for in the next piece
            if (c0 == 0 && task >= MOE_I8_NW && task + MOE_I8_NW < tasks) fetch(nxt, task + MOE_I8_NW);
#pragma unroll
            for (int s = 0; s < MOE_I8_DC; s++)
                if (s < cur.nu) acc = mi_mfma(cur.a[s], x[s], acc);
            if (used && c0 + (lane & 7) < n) {
                int *to = sums + ((sh ? L.P : 0) + row) * 8 + 4 * (lane >> 4 & 1);
#pragma unroll
                for (int i = 0; i < 4; i++) atomicAdd(to + i, acc[i]);   // integers: in any order the same
            }
        }
    };
    for (int task = wave; task < tasks; task += 2 * MOE_I8_NW) {
        piece(task, even, odd);
        if (task + MOE_I8_NW < tasks) piece(task + MOE_I8_NW, odd, even);
    }
    __syncthreads();
    // each sum becomes its weighted output, then a token's are added as k_moe_combine does: ascending expert id, then k;
    // then the shared experts
    for (int i = tid; i < rows * 8; i += MOE_I8_NT) {
        const int row = i >> 3, r = 8 * rb + (i & 7);
        const bool sh = row >= L.P;
        const int s = sh ? 0 : R.slot[row];
        if (s == MOE_I8_NONE) continue;
        const float ws = mi_float((i8_gp)(sh ? (const float *)L.sd.s0 : ts[s]), r);
        const float v = i8_out(sums[i], i8_get(L.hs + row), ws);
        sums[i] = __float_as_int(sh ? v : __fmul_rn(i8_weight(L, row, gen), v));
    }
    __syncthreads();
    for (int o = tid; o < L.T * 8; o += MOE_I8_NT) {
        const int t = o >> 3, ch = o & 7;
        float acc = 0.0f;
        for (int i = 0; i < L.K; i++) {
            const int p = order[t * L.K + i];
            if (R.slot[p] != MOE_I8_NONE) acc = __fadd_rn(acc, __int_as_float(sums[p * 8 + ch]));
        }
        if (L.shared) acc = __fadd_rn(acc, __int_as_float(sums[(L.P + t) * 8 + ch]));
        L.out[(size_t)t * L.H + 8 * rb + ch] = acc;
    }
}

__global__ __launch_bounds__(MOE_I8_NT, 4) void k_moe_i8(MoeI8Launch L) {
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ MoeI8Route R;
    const int b = blockIdx.x, gu = b - L.npre, sq = gu - L.ngu, rb = sq - L.nsq;
    const uint32_t next = (uint32_t)L.sync->gen[b] + 1u;
    const int gen = next ? next : 2;                           // 0: what was never set; 2: the halves of blocks keep their turns
    if (gu < 0) i8_pre(L, b, gen, lds);
    else if (sq < 0) i8_gate_up(L, gu, gen, R, lds);
    else if (rb < 0) i8_shared_codes(L, sq, gen, lds);
    else i8_down(L, rb, gen, R, lds);
    // the number of this launch, for all workgroups of the next, of which there may be more
    __syncthreads();
    for (int i = b + threadIdx.x * gridDim.x; i < MOE_I8_WGS; i += MOE_I8_NT * gridDim.x) L.sync->gen[i] = gen;
    if (b == 0)
        for (int i = threadIdx.x; i < MOE_I8_PAIRS; i += MOE_I8_NT) L.sync->blocks[~gen & 1][i] = 0;
}

// dynamic LDS of every role: gate+up's two buffers of sums
#define MOE_I8_LDS (2 * MOE_I8_NW * MOE_I8_RED * 16)
static_assert((MOE_I8_PAIRS + MOE_I8_TOK) * 32 + MOE_I8_PAIRS * 18 <= MOE_I8_LDS, "MoeI8Down");

// ================================================================================== host side
int run_moe_i8(bgl_ctx *c, const bgl_tensor *gate, const bgl_tensor *up, const bgl_tensor *down, const bgl_tensor *sg, const bgl_tensor *su,
               const bgl_tensor *sd, const float *rw, const float *rb, int renorm, const float *x, const int32_t *idx, const float *w, int T,
               int K, float *out) {
    MoeI8Launch L;
    memset(&L, 0, sizeof L);
    L.tg = (const BglDevTensor *)gate->dev_table; L.tu = (const BglDevTensor *)up->dev_table; L.td = (const BglDevTensor *)down->dev_table;
    L.shared = sg != nullptr;
    if (sg) { L.sg = sg->T; L.su = su->T; L.sd = sd->T; L.Ish = sg->T.N; }
    L.E = (int)gate->experts.size(); L.K = K; L.H = gate->T.K; L.I = gate->T.N;
    L.rw = rw; L.rb = rb; L.renorm = renorm;
    const int most = std::min(T, MOE_I8_TOK);
    // scratch of a chunk
    const size_t P = (size_t)most * K, rows = P + most;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t o = at; at += (bytes + 255) & ~(size_t)255; return o; };
    L.hp = (L.H + 127) & ~127; L.ip = (L.I + 127) & ~127; L.ishp = (L.Ish + 127) & ~127;
    const size_t o_hs = take(rows * 4), o_xs = take((size_t)most * 4), o_xq = take((size_t)most * L.hp), o_h = take(P * L.I * 4),
                 o_hsh = take((size_t)most * L.Ish * 4), o_hq = take(P * L.ip), o_hshq = take((size_t)most * L.ishp);
    if (dbuf_reserve(c, c->moe_g, at, false) || dbuf_reserve(c, c->moe_sync, sizeof(MoeI8Sync), true)) return bgl_last_code();
    L.sync = (MoeI8Sync *)c->moe_sync.p;
    uint8_t *base = (uint8_t *)c->moe_g.p;
    L.hs = (float *)(base + o_hs); L.xs = (float *)(base + o_xs); L.xq = (int8_t *)(base + o_xq);
    L.h = (float *)(base + o_h); L.hsh = (float *)(base + o_hsh); L.hq = (int8_t *)(base + o_hq); L.hshq = (int8_t *)(base + o_hshq);
    L.spin = c->mlp_spin;
    HIPCHK(hipFuncSetAttribute((const void *)k_moe_i8, hipFuncAttributeMaxDynamicSharedMemorySize, MOE_I8_LDS));
    for (int t0 = 0; t0 < T; t0 += MOE_I8_TOK) {
        L.T = std::min(MOE_I8_TOK, T - t0);
        L.P = L.T * K;
        L.nslots = std::min(L.E, L.P);
        L.x = x + (size_t)t0 * L.H;
        L.out = out + (size_t)t0 * L.H;
        L.idx = rw ? nullptr : idx + (size_t)t0 * K;
        L.w = rw ? nullptr : w + (size_t)t0 * K;
        L.never = c->mlp_test_timeout > 0 ? 1 : 0;                  // a test's launch, in which waits must give up
        if (c->mlp_test_timeout > 0) c->mlp_test_timeout--;
        L.npre = L.T + (rw ? L.T * ((L.E + MOE_I8_NW - 1) / MOE_I8_NW) : 0);
        L.ngu = std::min(MOE_I8_GU_WGS, (L.shared ? L.Ish / 16 : 0) + L.nslots * (L.I / 16));
        L.nsq = L.shared ? (L.T + MOE_I8_SQ - 1) / MOE_I8_SQ : 0;
        const int units = L.ip / 128, pieces = (units + MOE_I8_DC - 1) / MOE_I8_DC;      // of equal length
        L.piece = (units + pieces - 1) / pieces;
        const int tok = prof_begin(c, 1);
        hipLaunchKernelGGL(k_moe_i8, dim3((unsigned)(L.npre + L.ngu + L.nsq + L.H / 8)), dim3(MOE_I8_NT), MOE_I8_LDS, c->stream, L);
        prof_end(c, tok);
        HIPCHK(hipGetLastError());
    }
    return 0;
}
