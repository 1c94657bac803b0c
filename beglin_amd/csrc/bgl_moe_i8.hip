// bgl_moe_i8.hip -- a routed FFN (moe_ffn_batched, qwen_infer.c:5238-5350) of K_Q8C experts for a few tokens:
//
//   xq, xs = the int8 codes of each token          (k_moe_i8_pre, which also makes the router's scores)
//   g, u   = gate_e xq, up_e xq ; h = silu(g) * u   per pair (token, expert); the shared experts: per token
//   hq, hs = the int8 codes of each h row
//   out[t] = sum_e w_e * down_e hq (ascending expert ids) + shared down
//
// with the products of bgl_i8.hip (exact int32 sums, then fp32 operations in the order written there), so a
// row's bits depend neither on the other tokens nor on how the work is split.
//
// What bounds it is the experts' bytes: each touched expert is read once, whatever the number of its tokens
// (64 at the most; more go in chunks).
//   k_moe_i8_pre   the codes of x; the router's scores, a wave an expert, and the softmax and top-K of a token by
//                  whichever workgroup finishes its last score (a ticket per token; no workgroup waits)
//   k_moe_i8_gu    16-row blocks of both tensors of an expert and all of its tokens, in equal runs over two workgroups a
//                  CU, whose waves split K; the next block's weights are on their way while one is multiplied
//   k_moe_i8_hq    the codes of h, where a down workgroup would spend longer on making them all (MOE_I8_LDSQ)
//   k_moe_i8_down  a workgroup owns 16 output channels; its waves take pieces of the experts' K and add the int32 sums in
//                  LDS, which holds every pair's until the combine: no launch and no memory traffic for partial sums
// Workgroups find their expert and its pairs from the routing themselves.
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
#define MOE_I8_LDSQ (24 * 1024)   // h codes that a down workgroup makes for itself; more take a launch
#define MOE_I8_NW 8               // waves of a gate+up workgroup
#define MOE_I8_DW 16              // waves of a down workgroup
#define MOE_I8_DC 8               // units of 64 values that one of them takes at a time at most
#define MOE_I8_GU_WGS 512         // gate+up workgroups at most: two a CU

struct MoeI8Launch {
    const BglDevTensor *tg, *tu, *td;    // expert tables
    BglDevTensor sg, su, sd;             // shared experts (shared != 0)
    int shared, E, K, T, P, H, I, Ish, nslots, piece;   // nslots: the most slots; piece: units a down wave takes
    const float *x, *rw, *rb;            // token rows; router
    float *scores;                       // [T][E], null: idx / w are given
    int *ticket;                         // [T] workgroups of a token that have their scores; 0 between launches
    int renorm;
    int32_t *idx;                        // [P]
    float *w;
    int8_t *xq;
    float *xs;
    float *h, *hsh;                      // [P][I], [T][Ish]
    int8_t *hq, *hshq;                   // codes of h and their scales [P + T]; null: the down workgroups make them
    float *hs;
    float *out;
};

// ------------------------------------------------------------------ codes of x, routing
__global__ __launch_bounds__(256) void k_moe_i8_pre(MoeI8Launch L) {
    const int tid = threadIdx.x, lane = tid & 63;
    if ((int)blockIdx.x < L.T) {
        __shared__ uint32_t red[4];
        const int t = blockIdx.x;
        const float *x = L.x + (size_t)t * L.H;
        uint32_t mb = I8_MX0;
        for (int k = tid; k < L.H; k += 256) mb = max(mb, __float_as_uint(x[k]) & 0x7fffffffu);
        mb = wave_max_u32(mb);
        if (lane == 0) red[tid >> 6] = mb;
        __syncthreads();
        const I8Scale s = i8_scale(max(max(red[0], red[1]), max(red[2], red[3])));
        if (tid == 0) L.xs[t] = s.sc;
        for (int k = 4 * tid; k < L.H; k += 1024)
            *(uint32_t *)(L.xq + (size_t)t * L.H + k) = i8_pack4(i8_code(x[k], s), i8_code(x[k + 1], s), i8_code(x[k + 2], s), i8_code(x[k + 3], s));
        return;
    }
    // scores and ticket pass the L2s of the eight dies (agent scope), so no cache is written back for them: a score is in
    // memory before its workgroup's ticket is drawn, and who draws the last one reads them there
    const int per = (L.E + 3) / 4, b = blockIdx.x - L.T, t = b / per, e = (b % per) * 4 + (tid >> 6);
    __shared__ int last;
    __shared__ __align__(16) float lbuf[ROUTE_MAXE], sc[ROUTE_MAXE];
    if (e < L.E) {
        const double acc = route_dot_wave(L.rw + (size_t)e * L.H, L.x + (size_t)t * L.H, L.H, lane);
        const float s = L.rb ? __fadd_rn((float)acc, L.rb[e]) : (float)acc;
        if (lane == 0) __hip_atomic_store(L.scores + (size_t)t * L.E + e, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) last = __hip_atomic_fetch_add(L.ticket + t, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == per - 1;
    __syncthreads();
    if (!last || tid >= 64) return;
    for (int i = lane; i < L.E; i += 64)
        sc[i] = __hip_atomic_load(L.scores + (size_t)t * L.E + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (lane == 0) __hip_atomic_store(L.ticket + t, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next launch
    __builtin_amdgcn_wave_barrier();
    float sel_w[MOE_MAX_K];
    int sel_i[MOE_MAX_K];
    route_topk_wave(sc, L.E, L.K, L.renorm, lane, sel_i, sel_w, lbuf);
    if (lane == 0)
        for (int k = 0; k < L.K; k++) {
            L.idx[t * L.K + k] = sel_i[k];
            L.w[t * L.K + k] = sel_w[k];
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
__device__ __forceinline__ void i8_routing(const MoeI8Launch &L, MoeI8Route &R) {
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 63;
    if (tid < 32) R.used[tid] = 0;
    for (int s = tid; s < L.nslots; s += nt) R.at[s] = 0;
    __syncthreads();
    for (int p = tid; p < L.P; p += nt) {
        const int e = L.idx[p];
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
// a lane's operand address in block rb (16 rows) of a tensor, unit 0
__device__ __forceinline__ const uint8_t *mi_rows(const uint8_t *w, int cpr, int rb, int lane) {
    return w + ((size_t)(rb >> 2) * cpr + (lane >> 4)) * 1024 + ((rb & 3) * 16 + (lane & 15)) * 16;
}

// ------------------------------------------------------------------ gate + up
// h of the 16-row blocks rb0 .. rb1 - 1 for columns c0 .. of the n in list (a pair, or with list null a token): a wave
// takes every eighth unit of K, D at a time, and has the weights of the next D on their way while it multiplies.
template <int CB, int D>
__device__ __forceinline__ void i8_gu(const MoeI8Launch &L, const BglDevTensor &G, const BglDevTensor &Up, int rb0, int rb1, const uint16_t *list,
                                      int c0, int n, float *h, int width, i8_i4 *red) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int U = L.H / 64, NC = (U + D * MOE_I8_NW - 1) / (D * MOE_I8_NW), its = (rb1 - rb0) * NC;
    const int8_t *xp[CB];
#pragma unroll
    for (int j = 0; j < CB; j++) {
        const int c = min(c0 + 16 * j + (lane & 15), n - 1), tok = list ? list[c] / L.K : c;
        xp[j] = L.xq + (size_t)tok * L.H + (lane >> 4) * 16;
    }
    struct Ops { i8_u4 a[D], b[D]; } even, odd;                // in turn: no copy waits for a load
    auto load = [&](Ops &o, int it) {
        const int rb = rb0 + it / NC, u0 = (it % NC) * D * MOE_I8_NW + wave;
        const uint8_t *gp = mi_rows(G.w, G.cpr, rb, lane), *up = mi_rows(Up.w, Up.cpr, rb, lane);
#pragma unroll
        for (int s = 0; s < D; s++) {
            const int u = min(u0 + s * MOE_I8_NW, U - 1);
            o.a[s] = *(const i8_u4 *)(gp + (size_t)u * 4096);
            o.b[s] = *(const i8_u4 *)(up + (size_t)u * 4096);
        }
    };
    i8_i4 ga[CB], ua[CB];
    // the outputs that a thread forms, one for each NO: channel och of a block for column oc (a wave: 16 columns, 4 channels)
    constexpr int NO = CB <= 2 ? 1 : CB / 2;
    const int och = 4 * (wave & 3) + (lane & 3);
    int oc[NO], orow[NO];
    float xs[NO], gs, us;
#pragma unroll
    for (int i = 0; i < NO; i++) {
        oc[i] = c0 + 16 * ((wave >> 2) + 2 * i) + (lane >> 2);
        orow[i] = list ? list[min(oc[i], n - 1)] : min(oc[i], n - 1);
        xs[i] = L.xs[list ? orow[i] / L.K : orow[i]];
    }
    auto step = [&](int it, Ops &cur, Ops &nxt) {
        const int ch = it % NC, rb = rb0 + it / NC, u0 = ch * D * MOE_I8_NW + wave;
        i8_u4 x[D][CB];
#pragma unroll
        for (int s = 0; s < D; s++)
#pragma unroll
            for (int j = 0; j < CB; j++) x[s][j] = *(const i8_u4 *)(xp[j] + min(u0 + s * MOE_I8_NW, U - 1) * 64);
        if (ch == 0) {
#pragma unroll
            for (int j = 0; j < CB; j++) ga[j] = ua[j] = i8_i4{0, 0, 0, 0};
            gs = ((const float *)G.s0)[16 * rb + och];
            us = ((const float *)Up.s0)[16 * rb + och];
        }
        load(nxt, min(it + 1, its - 1));
#pragma unroll
        for (int s = 0; s < D; s++)
            if (u0 + s * MOE_I8_NW < U) {
#pragma unroll
                for (int j = 0; j < CB; j++) {
                    ga[j] = mi_mfma(cur.a[s], x[s][j], ga[j]);
                    ua[j] = mi_mfma(cur.b[s], x[s][j], ua[j]);
                }
            }
        if (ch != NC - 1) return;
        __syncthreads();                                       // an earlier block's sums have been read
#pragma unroll
        for (int j = 0; j < CB; j++) {
            red[((wave * CB + j) * 2) * 64 + lane] = ga[j];
            red[((wave * CB + j) * 2 + 1) * 64 + lane] = ua[j];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NO; i++) {
            const int j = (wave >> 2) + 2 * i;
            if (j >= CB) continue;
            const int *s = (const int *)red + j * 512 + (wave & 3) * 64 + lane;      // int (wave & 3) * 64 + lane of a block's 256
            int g = 0, u = 0;
#pragma unroll
            for (int w = 0; w < MOE_I8_NW; w++) {
                g += s[w * CB * 512];
                u += s[w * CB * 512 + 256];
            }
            if (oc[i] < n) h[(size_t)orow[i] * width + 16 * rb + och] = i8_swiglu(i8_out(g, xs[i], gs), i8_out(u, xs[i], us));
        }
    };
    load(even, 0);
    for (int it = 0; it < its; it += 2) {
        step(it, even, odd);
        if (it + 1 < its) step(it + 1, odd, even);
    }
}

// The 16-row blocks of the shared experts and then of each used expert, in equal runs over the workgroups.
template <int CB, int D>
__global__ __launch_bounds__(MOE_I8_NW * 64, 4) void k_moe_i8_gu(MoeI8Launch L) {
    extern __shared__ __align__(16) i8_i4 red[];               // [wave][column block][gate, up][64]
    __shared__ MoeI8Route R;
    i8_routing(L, R);
    const int nsh = L.shared ? L.Ish / 16 : 0, per = L.I / 16;
    const long all = nsh + (long)__builtin_amdgcn_readfirstlane(R.n) * per;
    const int end = (int)(all * (blockIdx.x + 1) / gridDim.x);
    for (int it = (int)(all * blockIdx.x / gridDim.x); it < end;) {
        const bool sh = it < nsh;
        const int slot = sh ? 0 : (it - nsh) / per, first = sh ? 0 : nsh + slot * per;    // (uniform)
        const int rb = it - first, rb1 = min(end - first, sh ? nsh : per);
        const int e = sh ? 0 : __builtin_amdgcn_readfirstlane((int)R.expert[slot]);
        const int l0 = sh ? 0 : __builtin_amdgcn_readfirstlane(R.off[slot]);
        const int n = sh ? L.T : __builtin_amdgcn_readfirstlane(R.off[slot + 1]) - l0;
        const BglDevTensor G = sh ? L.sg : L.tg[e], U = sh ? L.su : L.tu[e];
        const uint16_t *const list = sh ? nullptr : R.list + l0;
        float *const h = sh ? L.hsh : L.h;
        const int width = sh ? L.Ish : L.I;
        for (int c0 = 0; c0 < n; c0 += 16 * CB) i8_gu<CB, D>(L, G, U, rb, rb1, list, c0, n, h, width, red);
        it = first + rb1;
    }
}

// ------------------------------------------------------------------ codes of h where they take a launch
// A workgroup a row: rows [0, P) of I, then [0, T) of Ish.
__global__ __launch_bounds__(256) void k_moe_i8_hq(MoeI8Launch L) {
    __shared__ uint32_t red[4];
    const int tid = threadIdx.x, row = blockIdx.x;
    const bool sh = row >= L.P;
    const int width = sh ? L.Ish : L.I;
    const size_t at = (size_t)(sh ? row - L.P : row) * width;
    const float *h = (sh ? L.hsh : L.h) + at;
    uint32_t mb = I8_MX0;
    for (int k = 4 * tid; k < width; k += 1024) {
        const i8_f4 v = *(const i8_f4 *)(h + k);
#pragma unroll
        for (int i = 0; i < 4; i++) mb = max(mb, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    mb = wave_max_u32(mb);
    if ((tid & 63) == 0) red[tid >> 6] = mb;
    __syncthreads();
    const I8Scale s = i8_scale(max(max(red[0], red[1]), max(red[2], red[3])));
    if (tid == 0) L.hs[row] = s.sc;
    for (int k = 4 * tid; k < width; k += 1024) {
        const i8_f4 v = *(const i8_f4 *)(h + k);
        *(uint32_t *)((sh ? L.hshq : L.hq) + at + k) = i8_pack4(i8_code(v.x, s), i8_code(v.y, s), i8_code(v.z, s), i8_code(v.w, s));
    }
}

// ------------------------------------------------------------------ down + combine
template <bool LDSQ>
__global__ __launch_bounds__(MOE_I8_DW * 64) void k_moe_i8_down(MoeI8Launch L) {
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ MoeI8Route R;
    __shared__ const uint8_t *tw[MOE_I8_PAIRS];                          // each slot's weights and scales
    __shared__ const float *ts[MOE_I8_PAIRS];
    __shared__ uint16_t order[MOE_I8_PAIRS];
    __shared__ float hs[LDSQ ? MOE_I8_LDSQ / 64 : 1];                     // LDSQ: the scales of the rows (64 codes at least)
    int *const sums = (int *)dyn;                                        // [P + T][16]
    const int rows = L.P + (L.shared ? L.T : 0), tid = threadIdx.x;
    int8_t *const q = (int8_t *)dyn + (size_t)rows * 64;                 // LDSQ: the codes [P][I], [T][Ish]
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, rb = blockIdx.x;
    const int8_t *const hq = LDSQ ? q : L.hq, *const shq = LDSQ ? q + (size_t)L.P * L.I : L.hshq;
    for (int i = tid; i < rows * 16; i += MOE_I8_DW * 64) sums[i] = 0;
    i8_routing(L, R);
    const int nslots = __builtin_amdgcn_readfirstlane(R.n);
    for (int s = tid; s < nslots; s += MOE_I8_DW * 64) {
        tw[s] = L.td[R.expert[s]].w;
        ts[s] = (const float *)L.td[R.expert[s]].s0;
    }
    __syncthreads();
    // pieces of the shared experts first (the longest rows), then of the routed ones
    const int np = (L.I / 64 + L.piece - 1) / L.piece, nps = L.shared ? (L.Ish / 64 + L.piece - 1) / L.piece : 0;
    const int tasks = nps + nslots * np, cpr = (L.I + 127) / 128 * 8, scpr = (L.Ish + 127) / 128 * 8;
    struct Piece { int slot, u0, nu; i8_u4 a[MOE_I8_DC]; } even, odd;      // in turn: no copy waits for a load
    // a piece's place and weights
    auto fetch = [&](Piece &p, int task) {
        const bool sh = task < nps;
        p.slot = sh ? -1 : (task - nps) / np;
        p.u0 = (sh ? task : (task - nps) % np) * L.piece;
        p.nu = min(L.piece, (sh ? L.Ish : L.I) / 64 - p.u0);
        const uint8_t *wp = mi_rows(sh ? L.sd.w : tw[p.slot], sh ? scpr : cpr, rb, lane) + (size_t)p.u0 * 4096;
#pragma unroll
        for (int s = 0; s < MOE_I8_DC; s++) p.a[s] = *(const i8_u4 *)(wp + (size_t)min(s, p.nu - 1) * 4096);
    };
    if (wave < tasks) fetch(even, wave);                                 // on its way while the codes are made
    // a token's pairs by expert, then k: the order in which they are added
    for (int p = tid; p < L.P; p += MOE_I8_DW * 64) {
        const int t = p / L.K, me = R.slot[p];
        int before = 0;
        for (int o = t * L.K; o < (t + 1) * L.K; o++) before += R.slot[o] < me || (R.slot[o] == me && o < p);
        order[t * L.K + before] = (uint16_t)p;
    }
    if constexpr (LDSQ) {
        for (int row = wave; row < rows; row += MOE_I8_DW) {             // a wave a row
            const bool sh = row >= L.P;
            const int width = sh ? L.Ish : L.I;
            const float *h = sh ? L.hsh + (size_t)(row - L.P) * width : L.h + (size_t)row * width;
            int8_t *to = sh ? q + (size_t)L.P * L.I + (size_t)(row - L.P) * width : q + (size_t)row * width;
            uint32_t mb = I8_MX0;
            for (int k = 4 * lane; k < width; k += 256) {
                const i8_f4 v = *(const i8_f4 *)(h + k);
#pragma unroll
                for (int i = 0; i < 4; i++) mb = max(mb, __float_as_uint(v[i]) & 0x7fffffffu);
            }
            const I8Scale s = i8_scale(wave_max_u32(mb));
            if (lane == 0) hs[row] = s.sc;
            for (int k = 4 * lane; k < width; k += 256) {
                const i8_f4 v = *(const i8_f4 *)(h + k);
                *(uint32_t *)(to + k) = i8_pack4(i8_code(v.x, s), i8_code(v.y, s), i8_code(v.z, s), i8_code(v.w, s));
            }
        }
    }
    __syncthreads();
    auto piece = [&](int task, const Piece &cur, Piece &nxt) {
        const bool sh = cur.slot < 0;
        const int l0 = sh ? 0 : R.off[cur.slot], n = sh ? L.T : R.off[cur.slot + 1] - l0;
        const int8_t *const codes = (sh ? shq : hq) + cur.u0 * 64 + (lane >> 4) * 16;
        for (int c0 = 0; c0 < n; c0 += 16) {
            const int c = min(c0 + (lane & 15), n - 1), row = sh ? c : R.list[l0 + c];
            const int8_t *xp = codes + (size_t)row * (sh ? L.Ish : L.I);
            i8_i4 acc = {0, 0, 0, 0};
            i8_u4 x[MOE_I8_DC];
#pragma unroll
            for (int s = 0; s < MOE_I8_DC; s++) x[s] = *(const i8_u4 *)(xp + min(s, cur.nu - 1) * 64);
            // behind the codes: loads return in order, and these are waited for in the next piece
            if (c0 == 0 && task + MOE_I8_DW < tasks) fetch(nxt, task + MOE_I8_DW);
#pragma unroll
            for (int s = 0; s < MOE_I8_DC; s++)
                if (s < cur.nu) acc = mi_mfma(cur.a[s], x[s], acc);
            if (c0 + (lane & 15) < n) {
                int *to = sums + ((sh ? L.P : 0) + row) * 16 + 4 * (lane >> 4);
#pragma unroll
                for (int i = 0; i < 4; i++) atomicAdd(to + i, acc[i]);   // integers: in any order the same
            }
        }
    };
    for (int task = wave; task < tasks; task += 2 * MOE_I8_DW) {
        piece(task, even, odd);
        if (task + MOE_I8_DW < tasks) piece(task + MOE_I8_DW, odd, even);
    }
    __syncthreads();
    // each sum becomes its weighted output, then a token's are added as k_moe_combine does: ascending expert id, then k;
    // then the shared experts
    for (int i = tid; i < rows * 16; i += MOE_I8_DW * 64) {
        const int row = i >> 4, r = 16 * rb + (i & 15);
        const bool sh = row >= L.P;
        const int s = sh ? 0 : R.slot[row];
        if (s == MOE_I8_NONE) continue;
        const float ws = sh ? ((const float *)L.sd.s0)[r] : ts[s][r];
        const float v = i8_out(sums[i], LDSQ ? hs[row] : L.hs[row], ws);
        sums[i] = __float_as_int(sh ? v : __fmul_rn(L.w[row], v));
    }
    __syncthreads();
    for (int o = tid; o < L.T * 16; o += MOE_I8_DW * 64) {
        const int t = o >> 4, ch = o & 15;
        float acc = 0.0f;
        for (int i = 0; i < L.K; i++) {
            const int p = order[t * L.K + i];
            if (R.slot[p] != MOE_I8_NONE) acc = __fadd_rn(acc, __int_as_float(sums[p * 16 + ch]));
        }
        if (L.shared) acc = __fadd_rn(acc, __int_as_float(sums[(L.P + t) * 16 + ch]));
        L.out[(size_t)t * L.H + 16 * rb + ch] = acc;
    }
}

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
    const size_t o_hs = take(rows * 4), o_xs = take((size_t)most * 4), o_xq = take((size_t)most * L.H), o_h = take(P * L.I * 4),
                 o_hsh = take((size_t)most * L.Ish * 4), o_hq = take(P * L.I), o_hshq = take((size_t)most * L.Ish),
                 o_idx = take(P * 4), o_w = take(P * 4), o_sc = take((size_t)most * L.E * 4);
    if (dbuf_reserve(c, c->moe_g, at, false) || (rw && dbuf_reserve(c, c->moe_ticket, MOE_I8_TOK * 4, true))) return bgl_last_code();
    L.ticket = (int *)c->moe_ticket.p;
    uint8_t *base = (uint8_t *)c->moe_g.p;
    L.hs = (float *)(base + o_hs); L.xs = (float *)(base + o_xs); L.xq = (int8_t *)(base + o_xq);
    L.h = (float *)(base + o_h); L.hsh = (float *)(base + o_hsh);
    for (int t0 = 0; t0 < T; t0 += MOE_I8_TOK) {
        L.T = std::min(MOE_I8_TOK, T - t0);
        L.P = L.T * K;
        L.nslots = std::min(L.E, L.P);
        L.x = x + (size_t)t0 * L.H;
        L.out = out + (size_t)t0 * L.H;
        L.scores = rw ? (float *)(base + o_sc) : nullptr;
        L.idx = rw ? (int32_t *)(base + o_idx) : const_cast<int32_t *>(idx) + (size_t)t0 * K;
        L.w = rw ? (float *)(base + o_w) : const_cast<float *>(w) + (size_t)t0 * K;
        int tok = prof_begin(c, 2);
        hipLaunchKernelGGL(k_moe_i8_pre, dim3((unsigned)(L.T + (rw ? L.T * ((L.E + 3) / 4) : 0))), dim3(256), 0, c->stream, L);
        prof_end(c, tok);
        tok = prof_begin(c, 1);
        const unsigned wgs = (unsigned)std::min(MOE_I8_GU_WGS, (L.shared ? L.Ish / 16 : 0) + L.nslots * (L.I / 16));
        // Columns at a time: 2 blocks of 16 keep every register through the epilogue; 4 read a popular expert's weights once
        // instead of twice and keep less of them on their way.  64 experts of 2048 x 1408, 6 a token and a shared 2816:
        // 32 tokens 161 us with 2, 164 with 4; 64 tokens 214, 204.  (1 block runs into spills: 139 us for 129 at 16.)
        if (L.T <= 32) hipLaunchKernelGGL((k_moe_i8_gu<2, 2>), dim3(wgs), dim3(MOE_I8_NW * 64), MOE_I8_NW * 4096, c->stream, L);
        else hipLaunchKernelGGL((k_moe_i8_gu<4, 1>), dim3(wgs), dim3(MOE_I8_NW * 64), MOE_I8_NW * 8192, c->stream, L);
        const size_t q = (size_t)L.P * L.I + (size_t)(L.shared ? L.T * L.Ish : 0);
        const bool ldsq = q <= MOE_I8_LDSQ;
        L.hq = ldsq ? nullptr : (int8_t *)(base + o_hq);
        L.hshq = ldsq ? nullptr : (int8_t *)(base + o_hshq);
        if (!ldsq) hipLaunchKernelGGL(k_moe_i8_hq, dim3((unsigned)(L.P + (L.shared ? L.T : 0))), dim3(256), 0, c->stream, L);
        const int pieces = (L.I / 64 + MOE_I8_DC - 1) / MOE_I8_DC;            // of equal length
        L.piece = (L.I / 64 + pieces - 1) / pieces;
        const size_t lds = (size_t)(L.P + (L.shared ? L.T : 0)) * 64 + (ldsq ? q : 0);
        auto kern = ldsq ? k_moe_i8_down<true> : k_moe_i8_down<false>;
        HIPCHK(hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        hipLaunchKernelGGL(kern, dim3((unsigned)(L.H / 16)), dim3(MOE_I8_DW * 64), lds, c->stream, L);
        prof_end(c, tok);
        HIPCHK(hipGetLastError());
    }
    return 0;
}
