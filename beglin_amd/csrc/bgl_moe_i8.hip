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
// (64 at the most; more go in chunks).  A gate+up workgroup owns 16 rows of both tensors of one expert and all
// of its tokens, its waves splitting K; a down workgroup owns 16 output channels, its waves taking whole
// experts, and holds every pair's sum in LDS until the combine, so there is no launch and no memory traffic
// for partial sums.  Workgroups find their expert and its pairs from the routing themselves; up to
// MOE_I8_ROUTE tokens they also make it from the scores (softmax, top-K: about a microsecond a token and
// wave), so that a layer needs no launch for it.
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
#define MOE_I8_ROUTE 8            // up to this many tokens every workgroup makes the routing: one wave a token
#define MOE_I8_LDSQ (64 * 1024)   // h codes that a down workgroup makes for itself; more take a launch
#define MOE_I8_NW 8               // waves of a workgroup

struct MoeI8Launch {
    const BglDevTensor *tg, *tu, *td;    // expert tables
    BglDevTensor sg, su, sd;             // shared experts (shared != 0)
    int shared, E, K, T, P, H, I, Ish, nslots, parts;
    const float *x, *rw, *rb;            // token rows; router
    float *scores;                       // [T][E], null: idx / w are given
    int renorm;
    const int32_t *idx;                  // [P] where the scores are not routed by the workgroups
    const float *w;
    int8_t *xq;
    float *xs;
    float *h, *hsh;                      // [P][I], [T][Ish]
    uint32_t *amax;                      // [P + T] bits of the largest |h| of a row
    int8_t *hq, *hshq;                   // codes of h; null: the down workgroups make them
    float *out;
};

// ------------------------------------------------------------------ codes of x, scores, cleared maxima
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
        for (int k = tid; k < L.K; k += 256) L.amax[t * L.K + k] = 0;
        if (tid == 0) L.amax[L.P + t] = 0;
        return;
    }
    const int per = (L.E + 3) / 4, b = blockIdx.x - L.T, t = b / per, e = (b % per) * 4 + (tid >> 6);
    if (e >= L.E) return;
    const double acc = route_dot_wave(L.rw + (size_t)e * L.H, L.x + (size_t)t * L.H, L.H, lane);
    if (lane == 0) L.scores[(size_t)t * L.E + e] = L.rb ? __fadd_rn((float)acc, L.rb[e]) : (float)acc;
}

// ------------------------------------------------------------------ the routing in LDS
struct MoeI8Route {
    int ids[MOE_I8_PAIRS];               // expert of each pair
    float w[MOE_I8_PAIRS];
    uint32_t used[32];                   // experts that have a pair (E <= 1024)
};
__device__ __forceinline__ void i8_routing(const MoeI8Launch &L, MoeI8Route &R, float (*lbuf)[ROUTE_MAXE]) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (threadIdx.x < 32) R.used[threadIdx.x] = 0;
    if (!L.idx) {
        if (wave < L.T) route_topk_wave(L.scores + (size_t)wave * L.E, L.E, L.K, L.renorm, lane, R.ids + wave * L.K, R.w + wave * L.K, lbuf[wave]);
    } else {
        for (int p = threadIdx.x; p < L.P; p += blockDim.x) {
            R.ids[p] = L.idx[p];
            R.w[p] = L.w[p];
        }
    }
    __syncthreads();
    for (int p = threadIdx.x; p < L.P; p += blockDim.x) {
        const int e = R.ids[p];
        if (e >= 0 && e < L.E) atomicOr(&R.used[e >> 5], 1u << (e & 31));   // others are skipped
    }
    __syncthreads();
}
// the s-th used expert in ascending order (-1: there are fewer), by a whole wave
__device__ __forceinline__ int i8_slot(const MoeI8Route &R, int s) {
    const int lane = threadIdx.x & 63;
    const uint32_t word = lane < 32 ? R.used[lane] : 0u;
    int incl = __popc(word);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up(incl, o);
        if (lane >= o) incl += v;
    }
    const unsigned long long m = __ballot(incl > s);
    if (!m) return -1;
    const int l = __ffsll(m) - 1;
    uint32_t wd = __shfl(word, l);
    for (int left = s - (__shfl(incl, l) - __popc(wd)); left > 0; left--) wd &= wd - 1;
    return __builtin_amdgcn_readfirstlane(32 * l + __ffs(wd) - 1);
}
// the pairs of expert e in ascending order into list, by a whole wave; returns how many
__device__ __forceinline__ int i8_pairs(const MoeI8Launch &L, const MoeI8Route &R, int e, uint16_t *list) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int p0 = 0; p0 < L.P; p0 += 64) {
        const bool hit = p0 + lane < L.P && R.ids[p0 + lane] == e;
        const unsigned long long m = __ballot(hit);
        if (hit) list[n + __popcll(m & ((1ull << lane) - 1))] = (uint16_t)(p0 + lane);
        n += __popcll(m);
    }
    return n;
}

__device__ __forceinline__ i8_i4 mi_mfma(i8_u4 a, i8_u4 b, i8_i4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i8_i4, a), __builtin_bit_cast(i8_i4, b), c, 0, 0, 0);
}
// a lane's operand address in block rb (16 rows) of a tensor, unit 0
__device__ __forceinline__ const uint8_t *mi_rows(const uint8_t *w, int cpr, int rb, int lane) {
    return w + ((size_t)(rb >> 2) * cpr + (lane >> 4)) * 1024 + ((rb & 3) * 16 + (lane & 15)) * 16;
}

// ------------------------------------------------------------------ gate + up
// h of rows 16 rb .. + 15 for columns c0 .. of the n in list (a pair, or with list null a token)
template <int CB>
__device__ __forceinline__ void i8_gu(const MoeI8Launch &L, const BglDevTensor &G, const BglDevTensor &Up, int rb, const uint16_t *list, int c0,
                                      int n, float *h, int width, uint32_t *amax, i8_i4 *red) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int U = L.H / 64;
    const uint8_t *gp = mi_rows(G.w, G.cpr, rb, lane), *up = mi_rows(Up.w, Up.cpr, rb, lane);
    const int8_t *xp[CB];
#pragma unroll
    for (int j = 0; j < CB; j++) {
        const int c = min(c0 + 16 * j + (lane & 15), n - 1), tok = list ? list[c] / L.K : c;
        xp[j] = L.xq + (size_t)tok * L.H + (lane >> 4) * 16;
    }
    i8_i4 ga[CB], ua[CB];
#pragma unroll
    for (int j = 0; j < CB; j++) ga[j] = ua[j] = i8_i4{0, 0, 0, 0};
    constexpr int D = CB == 1 ? 4 : 2;
    for (int u0 = wave; u0 < U; u0 += D * MOE_I8_NW) {
        i8_u4 a[D], b[D], x[D][CB];
#pragma unroll
        for (int s = 0; s < D; s++) {
            const int u = min(u0 + s * MOE_I8_NW, U - 1);
            a[s] = *(const i8_u4 *)(gp + (size_t)u * 4096);
            b[s] = *(const i8_u4 *)(up + (size_t)u * 4096);
#pragma unroll
            for (int j = 0; j < CB; j++) x[s][j] = *(const i8_u4 *)(xp[j] + u * 64);
        }
#pragma unroll
        for (int s = 0; s < D; s++)
            if (u0 + s * MOE_I8_NW < U) {
#pragma unroll
                for (int j = 0; j < CB; j++) {
                    ga[j] = mi_mfma(a[s], x[s][j], ga[j]);
                    ua[j] = mi_mfma(b[s], x[s][j], ua[j]);
                }
            }
    }
    __syncthreads();                                   // an earlier chunk's sums have been read
#pragma unroll
    for (int j = 0; j < CB; j++) {
        red[((wave * CB + j) * 2) * 64 + lane] = ga[j];
        red[((wave * CB + j) * 2 + 1) * 64 + lane] = ua[j];
    }
    __syncthreads();
    for (int o = threadIdx.x; o < CB * 64; o += MOE_I8_NW * 64) {
        const int j = o >> 6, l = o & 63, c = c0 + 16 * j + (l & 15), r = 16 * rb + 4 * (l >> 4);
        uint32_t mb = 0;
        int row = 0;
        if (c < n) {
            i8_i4 g = {0, 0, 0, 0}, u = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < MOE_I8_NW; w++) {
                g += red[((w * CB + j) * 2) * 64 + l];
                u += red[((w * CB + j) * 2 + 1) * 64 + l];
            }
            row = list ? list[c] : c;
            const float xs = L.xs[list ? row / L.K : row];
            const i8_f4 gs = *(const i8_f4 *)((const float *)G.s0 + r), us = *(const i8_f4 *)((const float *)Up.s0 + r);
            i8_f4 v;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v[i] = i8_swiglu(i8_out(g[i], xs, gs[i]), i8_out(u[i], xs, us[i]));
                mb = max(mb, __float_as_uint(v[i]) & 0x7fffffffu);
            }
            *(i8_f4 *)(h + (size_t)row * width + r) = v;
        }
        mb = max(mb, (uint32_t)__shfl_xor((int)mb, 16));
        mb = max(mb, (uint32_t)__shfl_xor((int)mb, 32));
        if (c < n && l < 16) atomicMax(&amax[row], mb);      // a maximum: the order of the workgroups does not matter
    }
}

__global__ __launch_bounds__(MOE_I8_NW * 64, 4) void k_moe_i8_gu(MoeI8Launch L, int cbmax) {
    extern __shared__ __align__(16) i8_i4 red[];               // [wave][column block][gate, up][64]
    __shared__ MoeI8Route R;
    __shared__ __align__(16) float lbuf[MOE_I8_ROUTE][ROUTE_MAXE];
    __shared__ uint16_t list[MOE_I8_PAIRS];
    __shared__ int found[2];
    const int nsh = L.shared ? L.Ish / 16 : 0;
    BglDevTensor G, U;
    int rb, n;
    const uint16_t *ls = nullptr;
    float *h;
    int width;
    uint32_t *amax;
    if ((int)blockIdx.x < nsh) {
        G = L.sg; U = L.su; rb = blockIdx.x; n = L.T; h = L.hsh; width = L.Ish; amax = L.amax + L.P;
    } else {
        i8_routing(L, R, lbuf);
        const int b = blockIdx.x - nsh, per = L.I / 16;
        if (threadIdx.x < 64) {
            const int e = i8_slot(R, b / per), m = e < 0 ? 0 : i8_pairs(L, R, e, list);
            if (threadIdx.x == 0) { found[0] = e; found[1] = m; }
        }
        __syncthreads();
        const int e = __builtin_amdgcn_readfirstlane(found[0]);
        if (e < 0) return;
        n = __builtin_amdgcn_readfirstlane(found[1]);
        rb = b % per;
        G = L.tg[e]; U = L.tu[e]; ls = list; h = L.h; width = L.I; amax = L.amax;
    }
    for (int c0 = 0; c0 < n; c0 += 16 * cbmax) {
        const int left = n - c0;
        if (left <= 16 || cbmax == 1) i8_gu<1>(L, G, U, rb, ls, c0, n, h, width, amax, red);
        else if (left <= 32 || cbmax == 2) i8_gu<2>(L, G, U, rb, ls, c0, n, h, width, amax, red);
        else i8_gu<4>(L, G, U, rb, ls, c0, n, h, width, amax, red);
    }
}

// ------------------------------------------------------------------ codes of h where they take a launch
// Four values a thread; rows [0, P) of I, then [0, T) of Ish.  The maxima came with h.
__global__ __launch_bounds__(256) void k_moe_i8_hq(MoeI8Launch L) {
    const long q = (long)blockIdx.x * 256 + threadIdx.x, n0 = (long)L.P * L.I / 4;
    const bool sh = q >= n0;
    const long i = (sh ? q - n0 : q) * 4;
    const int width = sh ? L.Ish : L.I;
    if (sh && (!L.shared || i >= (long)L.T * L.Ish)) return;
    const int row = (int)(i / width);
    const I8Scale s = i8_scale(max(L.amax[(sh ? L.P : 0) + row], I8_MX0));
    const i8_f4 v = *(const i8_f4 *)((sh ? L.hsh : L.h) + i);
    *(uint32_t *)((sh ? L.hshq : L.hq) + i) = i8_pack4(i8_code(v.x, s), i8_code(v.y, s), i8_code(v.z, s), i8_code(v.w, s));
}

// ------------------------------------------------------------------ down + combine
// Sums of units [u0, u1) of 16 channels for columns c0 .. of the n rows (list, or row = column) of codes into LDS:
// sums[row * 16 + channel]
template <int CB, typename Rows>
__device__ __forceinline__ void i8_down(const uint8_t *wp, const int8_t *codes, int width, Rows rowof, int u0, int u1, int c0, int n, int *sums) {
    const int lane = threadIdx.x & 63;
    const int8_t *xp[CB];
#pragma unroll
    for (int j = 0; j < CB; j++) xp[j] = codes + (size_t)rowof(min(c0 + 16 * j + (lane & 15), n - 1)) * width + (lane >> 4) * 16;
    i8_i4 acc[CB];
#pragma unroll
    for (int j = 0; j < CB; j++) acc[j] = i8_i4{0, 0, 0, 0};
    constexpr int D = CB == 1 ? 8 : 4;
    for (int u = u0; u < u1; u += D) {
        i8_u4 a[D], x[D][CB];
#pragma unroll
        for (int s = 0; s < D; s++) {
            const int v = min(u + s, u1 - 1);
            a[s] = *(const i8_u4 *)(wp + (size_t)v * 4096);
#pragma unroll
            for (int j = 0; j < CB; j++) x[s][j] = *(const i8_u4 *)(xp[j] + v * 64);
        }
#pragma unroll
        for (int s = 0; s < D; s++)
            if (u + s < u1) {
#pragma unroll
                for (int j = 0; j < CB; j++) acc[j] = mi_mfma(a[s], x[s][j], acc[j]);
            }
    }
#pragma unroll
    for (int j = 0; j < CB; j++) {
        const int c = c0 + 16 * j + (lane & 15);
        if (c < n) *(i8_i4 *)(sums + rowof(c) * 16 + 4 * (lane >> 4)) = acc[j];
    }
}

template <bool LDSQ>
__global__ __launch_bounds__(MOE_I8_NW * 64) void k_moe_i8_down(MoeI8Launch L) {
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ MoeI8Route R;
    __shared__ __align__(16) float lbuf[MOE_I8_ROUTE][ROUTE_MAXE];
    __shared__ uint16_t lists[MOE_I8_NW][MOE_I8_PAIRS];
    int *const sums = (int *)dyn;                                        // [part][P + T][16]
    const int rows = L.P + (L.shared ? L.T : 0);
    int8_t *const q = (int8_t *)dyn + (size_t)L.parts * rows * 64;       // LDSQ: the codes [P][I], [T][Ish]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, rb = blockIdx.x;
    i8_routing(L, R, lbuf);
    if constexpr (LDSQ) {
        const int n0 = L.P * L.I / 4, n1 = n0 + (L.shared ? L.T * L.Ish / 4 : 0);
        for (int i = threadIdx.x; i < n1; i += MOE_I8_NW * 64) {
            const bool sh = i >= n0;
            const int at = (sh ? i - n0 : i) * 4, row = at / (sh ? L.Ish : L.I);
            const I8Scale s = i8_scale(max(L.amax[(sh ? L.P : 0) + row], I8_MX0));
            const i8_f4 v = *(const i8_f4 *)((sh ? L.hsh : L.h) + at);
            ((uint32_t *)q)[i] = i8_pack4(i8_code(v.x, s), i8_code(v.y, s), i8_code(v.z, s), i8_code(v.w, s));
        }
        __syncthreads();
    }
    const int8_t *const hq = LDSQ ? q : L.hq, *const shq = LDSQ ? q + (size_t)L.P * L.I : L.hshq;
    // the shared experts first (the longest rows), then the routed ones
    const int nsh = L.shared ? L.parts : 0;
    for (int task = wave; task < nsh + L.nslots * L.parts; task += MOE_I8_NW) {
        const bool sh = task < nsh;
        const int slot = sh ? 0 : (task - nsh) / L.parts, part = sh ? task : (task - nsh) % L.parts;
        const int e = sh ? 0 : i8_slot(R, slot);
        if (e < 0) break;                                                // slots past the last used expert
        const BglDevTensor *const T = sh ? &L.sd : L.td + e;
        const int n = sh ? L.T : i8_pairs(L, R, e, lists[wave]), width = sh ? L.Ish : L.I, U = width / 64;
        const uint8_t *wp = mi_rows(T->w, T->cpr, rb, lane);
        const int u0 = U * part / L.parts, u1 = U * (part + 1) / L.parts;
        int *const to = sums + (part * rows + (sh ? L.P : 0)) * 16;
        __builtin_amdgcn_wave_barrier();
        if (u0 == u1) {                                                  // fewer units than parts
            for (int i = lane; i < n * 16; i += 64) to[(sh ? i >> 4 : lists[wave][i >> 4]) * 16 + (i & 15)] = 0;
            continue;
        }
        for (int c0 = 0; c0 < n; c0 += 64) {
            const int left = n - c0;
            const uint16_t *ls = lists[wave];
            auto go = [&](auto rowof) {
                if (left <= 16) i8_down<1>(wp, sh ? shq : hq, width, rowof, u0, u1, c0, n, to);
                else if (left <= 32) i8_down<2>(wp, sh ? shq : hq, width, rowof, u0, u1, c0, n, to);
                else i8_down<4>(wp, sh ? shq : hq, width, rowof, u0, u1, c0, n, to);
            };
            if (sh) go([](int c) { return c; });
            else go([ls](int c) { return (int)ls[c]; });
        }
    }
    __syncthreads();
    // k_moe_combine's order: ascending expert id, then k; then the shared experts
    for (int o = threadIdx.x; o < L.T * 16; o += MOE_I8_NW * 64) {
        const int t = o >> 4, ch = o & 15, r = 16 * rb + ch;
        const int *ids = R.ids + t * L.K;
        auto value = [&](int row, const BglDevTensor *T) {
            int s = 0;
            for (int i = 0; i < L.parts; i++) s += sums[(i * rows + row) * 16 + ch];
            return i8_out(s, i8_scale(max(L.amax[row], I8_MX0)).sc, ((const float *)T->s0)[r]);
        };
        float acc = 0.0f;
        int last = -1, lastk = -1;                                        // the pair added last
        for (int a = 0; a < L.K; a++) {
            int be = 0x7fffffff, bk = -1;
            for (int k = 0; k < L.K; k++) {
                const int e = ids[k];
                if (e < 0 || e >= L.E) continue;
                if ((e > last || (e == last && k > lastk)) && e < be) { be = e; bk = k; }
            }
            if (bk < 0) break;
            acc = __fadd_rn(acc, __fmul_rn(R.w[t * L.K + bk], value(t * L.K + bk, L.td + be)));
            last = be;
            lastk = bk;
        }
        if (L.shared) acc = __fadd_rn(acc, value(L.P + t, &L.sd));
        L.out[(size_t)t * L.H + r] = acc;
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
    const size_t o_amax = take(rows * 4), o_xs = take((size_t)most * 4), o_xq = take((size_t)most * L.H), o_h = take(P * L.I * 4),
                 o_hsh = take((size_t)most * L.Ish * 4), o_hq = take(P * L.I), o_hshq = take((size_t)most * L.Ish),
                 o_idx = take(P * 4), o_w = take(P * 4), o_sc = take((size_t)most * L.E * 4);
    if (dbuf_reserve(c, c->moe_g, at, false)) return bgl_last_code();
    uint8_t *base = (uint8_t *)c->moe_g.p;
    L.amax = (uint32_t *)(base + o_amax); L.xs = (float *)(base + o_xs); L.xq = (int8_t *)(base + o_xq);
    L.h = (float *)(base + o_h); L.hsh = (float *)(base + o_hsh);
    for (int t0 = 0; t0 < T; t0 += MOE_I8_TOK) {
        L.T = std::min(MOE_I8_TOK, T - t0);
        L.P = L.T * K;
        L.nslots = std::min(L.E, L.P);
        L.x = x + (size_t)t0 * L.H;
        L.out = out + (size_t)t0 * L.H;
        L.scores = rw ? (float *)(base + o_sc) : nullptr;
        L.idx = rw ? nullptr : idx + (size_t)t0 * K;
        L.w = rw ? nullptr : w + (size_t)t0 * K;
        int tok = prof_begin(c, 2);
        hipLaunchKernelGGL(k_moe_i8_pre, dim3((unsigned)(L.T + (rw ? L.T * ((L.E + 3) / 4) : 0))), dim3(256), 0, c->stream, L);
        if (rw && L.T > MOE_I8_ROUTE) {
            bgl_launch_route_topk(L.scores, L.T, L.E, K, renorm, (int32_t *)(base + o_idx), (float *)(base + o_w), c->stream);
            L.idx = (const int32_t *)(base + o_idx);
            L.w = (const float *)(base + o_w);
        }
        prof_end(c, tok);
        tok = prof_begin(c, 1);
        const int cbmax = L.T <= 16 ? 1 : L.T <= 32 ? 2 : 4;
        hipLaunchKernelGGL(k_moe_i8_gu, dim3((unsigned)((L.shared ? L.Ish / 16 : 0) + L.nslots * (L.I / 16))), dim3(MOE_I8_NW * 64),
                           (size_t)MOE_I8_NW * cbmax * 2048, c->stream, L, cbmax);
        const size_t q = (size_t)L.P * L.I + (size_t)(L.shared ? L.T * L.Ish : 0);
        const bool ldsq = q <= MOE_I8_LDSQ;
        L.hq = ldsq ? nullptr : (int8_t *)(base + o_hq);
        L.hshq = ldsq ? nullptr : (int8_t *)(base + o_hshq);
        if (!ldsq) hipLaunchKernelGGL(k_moe_i8_hq, dim3((unsigned)((q / 4 + 255) / 256)), dim3(256), 0, c->stream, L);
        // few pairs: K is split as well, so that every wave has work
        L.parts = L.T == 1 ? 4 : L.T <= 4 ? 2 : 1;
        const size_t lds = (size_t)L.parts * (L.P + (L.shared ? L.T : 0)) * 64 + (ldsq ? q : 0);
        auto kern = ldsq ? k_moe_i8_down<true> : k_moe_i8_down<false>;
        HIPCHK(hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        hipLaunchKernelGGL(kern, dim3((unsigned)(L.H / 16)), dim3(MOE_I8_NW * 64), lds, c->stream, L);
        prof_end(c, tok);
        HIPCHK(hipGetLastError());
    }
    return 0;
}
