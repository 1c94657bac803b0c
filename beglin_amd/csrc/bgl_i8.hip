// bgl_i8.hip -- products of int8 codes with one scale per token and per output channel (BGL_K_Q8C):
//
//   y[m][r] = (float)(sum_c xq[m][c] * wq[r][c]) * (xs[m] * ws[r]) + bias[r]
//
// The sum is an int32 and exact, so neither its order nor a split of K changes a bit: waves may take any
// share of K.  The device layout is that of int8 group-64 tensors ([64-row tile][16-byte chunk][row]), K
// padded to 128 with zero codes: four chunks of 16 rows are the A operand of v_mfma_i32_16x16x64_i8 as
// they lie in memory (lane l: row l % 16, values 16 (l / 16) .. + 15), the codes of a token row are its B
// operand, and a lane's four results are four neighbouring channels of one token.  The zero padding of
// the weights also means that what an activation row holds past K never counts.
#include <string.h>

#include <algorithm>

#include "../../include/beglin_qgemv.h"
#include "bgl_i8.h"

#define HIPCHK(expr)                                                                             \
    do {                                                                                         \
        hipError_t e_ = (expr);                                                                  \
        if (e_ != hipSuccess) return bgl_fail(BGL_E_HIP, "%s: %s", #expr, hipGetErrorString(e_)); \
    } while (0)

struct I8Task {
    BglDevTensor T;
    const float *bias;
    void *y;
    long ldy;
    int blk0;                 // first workgroup row block of this tensor
    int *part;                // K split: the slices' sums [slice][M][N rounded up to 4], joined by k_i8_join
};
struct I8Launch {
    I8Task t[BGL_MAX_TASKS];
    int glu;                      // t[0] and t[1] are gate and up of one h = silu(gate x) * up x, written to t[0].y
    int ks;                       // slices of K (grid z); 1: the outputs are written at once
    int n, M, K16, y_type;        // K16: K rounded up to 16
    const int8_t *xq;
    long ldq;
    const float *xs;
    const float *xf;              // the columns before quantization, [M][K]: each workgroup makes the codes it needs; or null
    float *xs_out;                // then K split: where their scales go
};

__device__ __forceinline__ i8_i4 i8_mfma(i8_u4 a, i8_u4 b, i8_i4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i8_i4, a), __builtin_bit_cast(i8_i4, b), c, 0, 0, 0);
}

// The workgroup's tensor, picked by selects so that its fields come in one round of scalar loads.
__device__ __forceinline__ I8Task i8_task(const I8Launch &L, int blk) {
    I8Task t = L.t[0];
#pragma unroll
    for (int i = 1; i < BGL_MAX_TASKS; i++)
        if (i < L.n && blk >= L.t[i].blk0) t = L.t[i];
    return t;
}

// Four outputs of a lane in one store, wherever their row begins (gfx950 stores 8 and 16 bytes at any address; as single
// values the outputs of 3101 x 8030 x 523, whose rows begin off 8 bytes, took 64 us in all, 42 so).
typedef float i8_sf4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned int i8_su2 __attribute__((ext_vector_type(2), aligned(2)));
// Four neighbouring channels r .. r + 3 of token m.
__device__ __forceinline__ void i8_store4(const I8Launch &L, const I8Task &t, int m, int r, i8_i4 acc, float as, i8_f4 ws, i8_f4 b) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = i8_out(acc[i], as, ws[i]);
    if (t.bias) {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __fadd_rn(v[i], b[i]);
    }
    const size_t at = (size_t)m * t.ldy + r;
    if (r + 4 <= t.T.N) {
        if (L.y_type == BGL_T_F32) *(i8_sf4 *)((float *)t.y + at) = i8_sf4{v[0], v[1], v[2], v[3]};
        else
            *(i8_su2 *)((uint16_t *)t.y + at) = i8_su2{(uint32_t)i8_h16(v[0], L.y_type) | ((uint32_t)i8_h16(v[1], L.y_type) << 16),
                                                       (uint32_t)i8_h16(v[2], L.y_type) | ((uint32_t)i8_h16(v[3], L.y_type) << 16)};
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (r + i < t.T.N) i8_st(t.y, L.y_type, at + i, v[i]);
    }
}
__device__ __forceinline__ int i8_np(int N) { return (N + 3) & ~3; }
// scales (the device copy is padded to whole tiles) and biases of channels r .. r + 3
__device__ __forceinline__ i8_f4 i8_ws(const I8Task &t, int r) { return *(const i8_f4 *)((const float *)t.T.s0 + r); }
__device__ __forceinline__ i8_f4 i8_bias(const I8Task &t, int r) {
    i8_f4 b = {0.0f, 0.0f, 0.0f, 0.0f};
    if (t.bias) {
#pragma unroll
        for (int i = 0; i < 4; i++) b[i] = t.bias[min(r + i, t.T.N - 1)];
    }
    return b;
}

// ================================================================================== few columns
// A workgroup owns RB blocks of 16 channels and up to 16 CB tokens; its waves split K.  F32: the tokens come in fp32, and
// every workgroup makes their codes in LDS (bgl_norm.hip's arithmetic) while its first weights are on their way.  Weights and codes
// go straight from memory to the operand registers, D units ahead; the waves' int32 sums meet in LDS.
// Partial sums of at most I8_S_PART / (RB * CB) waves lie in LDS at once: a workgroup of twice that many waves first
// adds the upper half's to the lower half's.
#define I8_S_PART 64          // KB
#define I8_S_RND 4            // F32: 4 values a thread this often at most
template <int RB, int CB>
constexpr int i8_s_waves() { return RB * CB <= 4 ? 16 : 8; }
template <int RB, int CB, int D, bool F32, bool GLU>
__global__ __launch_bounds__((i8_s_waves<RB, CB>() * 64)) void k_i8_s(I8Launch L) {
    extern __shared__ __align__(16) i8_i4 red[];               // [wave][RB * CB][64]; F32: codes [M][K + 16], a word a column
    constexpr int Q = RB * CB, G = I8_S_PART / Q;
    const int nw = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    constexpr int RP = GLU ? RB / 2 : RB;
    const I8Task t = GLU ? L.t[0] : i8_task(L, blockIdx.x);
    const int m0 = blockIdx.y * 64;
    const int rb0 = (blockIdx.x - t.blk0) * RP;                     // RP divides 4: the blocks lie in one tile
    const int U0 = t.T.nunits * blockIdx.z / L.ks, U = t.T.nunits * (blockIdx.z + 1) / L.ks;
    const size_t wo = ((size_t)(rb0 >> 2) * t.T.cpr + (lane >> 4)) * 1024 + ((rb0 & 3) * 16 + (lane & 15)) * 16;
    const uint8_t *wp = t.T.w + wo, *wu = GLU ? L.t[1].T.w + wo : nullptr;
    const int8_t *xp[CB];
    const int kq = (lane >> 4) * 16;
    int8_t *const codes = (int8_t *)(red + min(nw * Q, I8_S_PART) * 64);
    uint32_t *const mx = (uint32_t *)(codes + L.M * (t.T.K + 16));
    const int grp = nw * 4, per = t.T.K / 64, nch = F32 ? L.M * per : 0;
    i8_f4 xv[I8_S_RND];
    if constexpr (F32) {
        // 16 lanes take 64 values of a column; these loads go out before the weights, which need not be there for the codes
#pragma unroll
        for (int r = 0; r < I8_S_RND; r++)
            if (r * grp < nch) xv[r] = *(const i8_f4 *)(L.xf + (size_t)min(r * grp + (int)(threadIdx.x >> 4), nch - 1) * 64 + 4 * (threadIdx.x & 15));
        if (threadIdx.x < L.M) mx[threadIdx.x] = I8_MX0;
        xp[0] = codes + min(lane & 15, L.M - 1) * (t.T.K + 16);
    } else
#pragma unroll
    for (int j = 0; j < CB; j++) xp[j] = L.xq + (size_t)min(m0 + 16 * j + (lane & 15), L.M - 1) * L.ldq;
    i8_i4 acc[RB][CB];
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int j = 0; j < CB; j++) acc[i][j] = i8_i4{0, 0, 0, 0};
    struct Ops { i8_u4 a[D][RB], b[D][CB]; } even, odd;             // in turn: no copy waits for a load
    auto load = [&](Ops &o, int u0) {
#pragma unroll
        for (int s = 0; s < D; s++) {
            const int u = min(u0 + s * nw, U - 1);
#pragma unroll
            for (int i = 0; i < RB; i++) o.a[s][i] = *(const i8_u4 *)((i < RP ? wp : wu) + (size_t)u * 4096 + 256 * (i % RP));
            const int k = min(64 * u + kq, L.K16 - 16);              // past the row: the weights are zero there
#pragma unroll
            for (int j = 0; j < CB; j++)
                if (!F32) o.b[s][j] = *(const i8_u4 *)(xp[j] + k);
        }
    };
    auto step = [&](int u0, const Ops &cur, Ops &nxt) {
        if (u0 + D * nw < U) load(nxt, u0 + D * nw);
#pragma unroll
        for (int s = 0; s < D; s++) {
            if (u0 + s * nw < U) {
                if constexpr (F32) {
                    const i8_u4 b = *(const i8_u4 *)(xp[0] + min(64 * (u0 + s * nw) + kq, L.K16 - 16));
#pragma unroll
                    for (int i = 0; i < RB; i++) acc[i][0] = i8_mfma(cur.a[s][i], b, acc[i][0]);
                    continue;
                }
#pragma unroll
                for (int i = 0; i < RB; i++)
#pragma unroll
                    for (int j = 0; j < CB; j++) acc[i][j] = i8_mfma(cur.a[s][i], cur.b[s][j], acc[i][j]);
            }
        }
    };
    load(even, U0 + wave);
    if constexpr (F32) {
        __syncthreads();
#pragma unroll
        for (int r = 0; r < I8_S_RND; r++) {
            if (r * grp >= nch) break;
            uint32_t mb = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) mb = max(mb, __float_as_uint(xv[r][i]) & 0x7fffffffu);
            mb = max(mb, (uint32_t)dpp_i<0xB1>((int)mb));
            mb = max(mb, (uint32_t)dpp_i<0x4E>((int)mb));
            mb = max(mb, (uint32_t)dpp_i<0x141>((int)mb));
            mb = max(mb, (uint32_t)dpp_i<0x140>((int)mb));
            if ((threadIdx.x & 15) == 0) atomicMax(&mx[min(r * grp + (int)(threadIdx.x >> 4), nch - 1) / per], mb);
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < I8_S_RND; r++) {
            const int ch = r * grp + (threadIdx.x >> 4);
            if (ch >= nch) break;
            const int m = ch / per;
            const I8Scale s = i8_scale(mx[m]);
            *(uint32_t *)(codes + m * (t.T.K + 16) + (ch - m * per) * 64 + 4 * (threadIdx.x & 15)) =
                i8_pack4(i8_code(xv[r].x, s), i8_code(xv[r].y, s), i8_code(xv[r].z, s), i8_code(xv[r].w, s));
        }
        if (L.ks > 1 && blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x < L.M) L.xs_out[threadIdx.x] = i8_scale(mx[threadIdx.x]).sc;
        __syncthreads();
    }
    for (int u0 = U0 + wave; u0 < U; u0 += 2 * D * nw) {
        step(u0, even, odd);
        if (u0 + D * nw < U) step(u0 + D * nw, odd, even);
    }
    auto put = [&](int at) {
#pragma unroll
        for (int i = 0; i < RB; i++)
#pragma unroll
            for (int j = 0; j < CB; j++) red[(at * Q + i * CB + j) * 64 + lane] = acc[i][j];
    };
    if (i8_s_waves<RB, CB>() > G && nw > G) {
        if (wave >= G) put(wave - G);
        __syncthreads();
        if (wave < nw - G) {
#pragma unroll
            for (int i = 0; i < RB; i++)
#pragma unroll
                for (int j = 0; j < CB; j++) acc[i][j] += red[(wave * Q + i * CB + j) * 64 + lane];
        }
        __syncthreads();
    }
    if (wave < G) put(wave);
    __syncthreads();
    const int parts = min(nw, G);
    for (int o = threadIdx.x; o < RP * CB * 64; o += blockDim.x) {
        const int l = o & 63, j = (o >> 6) % CB, i = (o >> 6) / CB;
        const int m = m0 + 16 * j + (l & 15), r = (rb0 + i) * 16 + 4 * (l >> 4);
        if (m >= L.M || r >= t.T.N) continue;
        i8_i4 s = {0, 0, 0, 0};
        for (int w = 0; w < parts; w++) s += red[(w * Q + i * CB + j) * 64 + l];
        if constexpr (GLU) {
            i8_i4 s2 = {0, 0, 0, 0};
            for (int w = 0; w < parts; w++) s2 += red[(w * Q + (i + RP) * CB + j) * 64 + l];
            const float as = F32 ? i8_scale(mx[m]).sc : L.xs[m];
            const i8_f4 gs = i8_ws(t, r), us = i8_ws(L.t[1], r);
            i8_f4 h;
#pragma unroll
            for (int e = 0; e < 4; e++) h[e] = i8_swiglu(i8_out(s[e], as, gs[e]), i8_out(s2[e], as, us[e]));
            float *y = (float *)t.y + (size_t)m * t.ldy + r;
            if (r + 4 <= t.T.N) *(i8_sf4 *)y = i8_sf4{h[0], h[1], h[2], h[3]};
            else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (r + e < t.T.N) y[e] = h[e];
            }
        } else if (L.ks > 1) *(i8_i4 *)(t.part + ((size_t)blockIdx.z * L.M + m) * i8_np(t.T.N) + r) = s;
        else i8_store4(L, t, m, r, s, F32 ? i8_scale(mx[m]).sc : L.xs[m], i8_ws(t, r), i8_bias(t, r));
    }
}

// ================================================================================== many columns
// Tiles of 16 CM NWM tokens by 16 CN NWN channels (128 x 128, 128 x 192, 256 x 256), NWM x NWN waves; both operands go through LDS in
// two stages of 128 values of K, copied there without passing through registers (buffer loads to LDS).  A wave reads
// the operands of half a stage from LDS while it multiplies the half before, so that its products wait neither for
// LDS nor at the barrier, of which there is one a stage: between the halves, when every wave has read the whole stage
// and the next one has landed; the copies of the stage after that go out among the products that follow.
//
// A stage of weights keeps the device layout ([64-row tile][chunk][row], 1 KB runs).  A stage of token
// rows is [row][128 bytes] with chunk c of row r at place c ^ (r / 2 % 8): an instruction copies 8 whole
// rows, and the 16 rows that an operand read touches lie in different banks (none in conflict, by the counters).  Stages
// of 64 values, four of them, took as long for the copies alone as the products do: a copy of 64-byte pieces of 16 rows
// moves half of what one of 128-byte pieces does (4096 x 4096 x 14336: 206 us so, 190 now).
//
// 256 x 256 tiles: 8192 x 8192 x 8192 in 438 us, 2.51 POP/s (the library's int8 product: 474 us); a wave's products
// without copies and reads would take 262 us at the clock that the card holds there (2.0 GHz).
typedef unsigned int i8_rsrc __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i8_rsrc i8_mkrsrc(const void *p, uint32_t bytes) {
    const uint64_t a = (uint64_t)(uintptr_t)p;
    i8_rsrc r;
    r.x = __builtin_amdgcn_readfirstlane((uint32_t)a);
    r.y = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xffffu);
    r.z = __builtin_amdgcn_readfirstlane(bytes);
    r.w = 0x00020000u;
    return r;
}
// 64 lanes x 16 bytes at rsrc + voff + soff into LDS at lds + 16 * lane.  Written as asm because the compiler
// would wait for every copy in flight before each LDS read; i8_wait below is the wait that counts.  (m0 is
// never live across code of the compiler's: it sets m0 right before an instruction that reads it.)
__device__ __forceinline__ void i8_copy(i8_rsrc rs, uint32_t voff, uint32_t soff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(voff), "s"(rs), "s"(soff)
                 : "memory");
}
// Every copy of each wave has landed and every LDS read of it has returned.  (The barrier alone is no access to memory for
// the compiler: the empty asm behind it keeps later reads from moving before it.)
__device__ __forceinline__ void i8_wait() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Workgroup b of nt: each XCD (workgroups go round the 8 of them) takes a run of neighbouring tiles, and
// within it 8 tiles of tokens share the weights that they read from its L2.
__device__ __forceinline__ void i8_tile(int b, int ntm, int ntn, int &tm, int &tn) {
    const int nt = ntm * ntn, x = b & 7, q = nt >> 3, rem = nt & 7;
    const int id = x * q + min(x, rem) + (b >> 3);
    const int gw = 8 * ntn, g = id / gw, in = id % gw, gm = min(8, ntm - 8 * g);
    tm = 8 * g + in % gm;
    tn = in / gm;
}

template <int CM, int CN, int NWM, int NWN>
__global__ __launch_bounds__(NWM *NWN * 64, 2) void k_i8_l(I8Launch L, int ntm, int ntn) {
    constexpr int BK = 128, BM = 16 * CM * NWM, BN = 16 * CN * NWN, NW = NWM * NWN;
    constexpr int XB = BM * BK, WB = BN * BK, SB = XB + WB;                   // bytes of a stage
    constexpr int XI = XB / 1024 / NW, WI = WB / 1024 / NW;                   // copies of a wave per stage
    static_assert(XI * NW * 1024 == XB && WI * NW * 1024 == WB && BN % 64 == 0, "whole copies");
    extern __shared__ __align__(1024) uint8_t sm[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    int tm, tn;
    i8_tile(blockIdx.x, ntm, ntn, tm, tn);
    const I8Task t = i8_task(L, tn);
    const int m0 = tm * BM, n0 = (tn - t.blk0) * BN;
    const int all = t.T.nunits / 2, s0 = all * blockIdx.z / L.ks, ns = all * (blockIdx.z + 1) / L.ks;   // K is padded to whole stages
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)sm;

    // token rows: copy j of the stage is rows 8 j .. 8 j + 7; rows past M repeat the last one
    const int rows = min(BM, L.M - m0);
    const i8_rsrc xr = i8_mkrsrc(L.xq + (size_t)m0 * L.ldq, (uint32_t)((rows - 1) * L.ldq + L.K16));
    uint32_t xo[XI];
#pragma unroll
    for (int i = 0; i < XI; i++) {
        const int r = 8 * (wave + NW * i) + (lane >> 3);
        xo[i] = (uint32_t)(min(r, rows - 1) * (int)L.ldq + (((lane & 7) ^ ((r >> 1) & 7)) << 4));
    }
    // weights: copy j is chunk j % 8 of tile j / 8; tiles past the tensor's last repeat it
    const int tile0 = n0 / 64, tb = t.T.cpr * 1024;
    const i8_rsrc wr = i8_mkrsrc(t.T.w + (size_t)tile0 * tb, (uint32_t)(min(BN / 64, t.T.ntiles - tile0) * tb));
    uint32_t wo[WI];
#pragma unroll
    for (int i = 0; i < WI; i++) {
        const int j = wave + NW * i;
        wo[i] = (uint32_t)(min(j >> 3, t.T.ntiles - 1 - tile0) * tb + (j & 7) * 1024);
    }
    auto copy = [&](int i, int s, uint32_t base) {                            // the wave's i-th copy of stage s
        if (i < WI) i8_copy(wr, lane * 16, wo[i] + s * 8192, base + (wave + NW * i) * 1024);
        else i8_copy(xr, xo[i - WI] + s * BK, 0, base + WB + (wave + NW * (i - WI)) * 1024);
    };
    const int wm = wave / NWN, wn = wave % NWN;
    i8_i4 acc[CM][CN];
#pragma unroll
    for (int i = 0; i < CM; i++)
#pragma unroll
        for (int j = 0; j < CN; j++) acc[i][j] = i8_i4{0, 0, 0, 0};
    // a lane's operand addresses in a stage, for each of its halves of 64 values
    const int key = (lane & 15) >> 1, xl = WB + (wm * CM * 16 + (lane & 15)) * BK;
    const int xh[2] = {xl + (((lane >> 4) ^ key) << 4), xl + (((4 + (lane >> 4)) ^ key) << 4)};
    const int wl = (lane >> 4) * 1024 + (lane & 15) * 16;
    i8_u4 a[2][CN], b[2][CM];
    auto ld_a = [&](int h, int j, const uint8_t *st) {
        const int nb = wn * CN + j;
        a[h][j] = *(const i8_u4 *)(st + (nb >> 2) * 8192 + (nb & 3) * 256 + h * 4096 + wl);
    };
    auto ld_b = [&](int h, int i, const uint8_t *st) { b[h][i] = *(const i8_u4 *)(st + xh[h] + i * 16 * BK); };
    // The products of half h, with the operands of the other half (of the stage at st) read among them, and with
    // `from` the copies of stage s into the stage at base.
    auto half = [&](int h, const uint8_t *st, bool more, int s, uint32_t base) {
#pragma unroll
        for (int i = 0; i < CM; i++) {
#pragma unroll
            for (int j = i * CN / CM; j < (i + 1) * CN / CM; j++) ld_a(h ^ 1, j, st);
            ld_b(h ^ 1, i, st);
#pragma unroll
            for (int j = 0; j < CN; j++) acc[i][j] = i8_mfma(a[h][j], b[h][i], acc[i][j]);
            if (more) {
#pragma unroll
                for (int q = i * (WI + XI) / CM; q < (i + 1) * (WI + XI) / CM; q++) copy(q, s, base);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
#pragma unroll
    for (int q = 0; q < WI + XI; q++) copy(q, s0, lds0);
    i8_wait();
    if (s0 + 1 < ns) {
#pragma unroll
        for (int q = 0; q < WI + XI; q++) copy(q, s0 + 1, lds0 + SB);
    }
#pragma unroll
    for (int j = 0; j < CN; j++) ld_a(0, j, sm);
#pragma unroll
    for (int i = 0; i < CM; i++) ld_b(0, i, sm);
    uint32_t cur = 0;                                                         // the stage that is multiplied: 0 or SB
    for (int s = s0; s < ns; s++) {
        half(0, sm + cur, false, 0, 0);
        // every wave has read the whole stage, and the next one has landed: it is read while this one's place is filled
        i8_wait();
        half(1, sm + (SB - cur), s + 2 < ns, s + 2, lds0 + cur);              // (the last stage reads what lies there)
        cur = SB - cur;
    }
    // a token's channels one after the other: the pieces of a line meet in the L2 (the other way round 4096 x 14336 bf16
    // outputs were 224 MB of writes, and are their 117 so: 270 us -> 242)
    i8_f4 ws[CN], bias[CN];
#pragma unroll
    for (int j = 0; j < CN; j++) {
        const int r = min(n0 + (wn * CN + j) * 16 + 4 * (lane >> 4), t.T.ntiles * 64 - 4);
        ws[j] = i8_ws(t, r);
        bias[j] = i8_bias(t, r);
    }
#pragma unroll
    for (int i = 0; i < CM; i++) {
        const int m = m0 + (wm * CM + i) * 16 + (lane & 15);
        if (m >= L.M) continue;
        const float as = L.ks > 1 ? 0.0f : L.xs[m];
#pragma unroll
        for (int j = 0; j < CN; j++) {
            const int r = n0 + (wn * CN + j) * 16 + 4 * (lane >> 4);
            if (r >= t.T.N) continue;
            if (L.ks > 1) *(i8_i4 *)(t.part + ((size_t)blockIdx.z * L.M + m) * i8_np(t.T.N) + r) = acc[i][j];
            else i8_store4(L, t, m, r, acc[i][j], as, ws[j], bias[j]);
        }
    }
}

// The slices' sums added (integers: in any order the same) and the outputs written, four channels a thread.
__global__ __launch_bounds__(256) void k_i8_join(I8Launch L) {
    const I8Task t = i8_task(L, blockIdx.z);                   // (blk0 holds the tensor's place in the group)
    const int np = i8_np(t.T.N), r = (blockIdx.x * 256 + threadIdx.x) * 4, m = blockIdx.y;
    if (r >= np) return;
    const size_t slice = (size_t)L.M * np;
    const int *p = t.part + (size_t)m * np + r;
    i8_i4 s = {0, 0, 0, 0};
#pragma unroll 4
    for (int z = 0; z < L.ks; z++) s += *(const i8_i4 *)(p + z * slice);
    i8_store4(L, t, m, r, s, L.xs[m], i8_ws(t, r), i8_bias(t, r));
}

// ================================================================================== host side
#define I8_CUS 256
#define I8_SLICE 512          // values of K that a slice has at least
#define I8_JOIN 3.2e6         // bytes of slices' sums that are written and joined in a us
// Room for the slices' sums, the same for every call that could split K at its or at fewer columns, so that those may
// be captured after it.  A choice that does not fit (many columns in many slices, which would cost more than they give)
// keeps K whole.
#define I8_PART_BYTES ((size_t)32 << 20)

static size_t i8_part(const I8Launch &L, int ks) {
    size_t v = 0;
    for (int i = 0; i < L.n; i++) v += (size_t)ks * L.M * ((L.t[i].T.N + 3) & ~3) * 4;
    return v;
}
// Points the tensors at their slices' sums; with no room for them (the no-alloc entry's fixed scratch) K stays whole.
static int i8_split(bgl_ctx *c, I8Launch &L, int ks) {
    L.ks = 1;
    const int units = L.t[0].T.nunits;
    if (units * 64 < 2 * I8_SLICE) return 0;
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    if (!c->fixed_base) HIPCHK(hipStreamIsCapturing(c->stream, &cs));
    if (!c->fixed_base && cs == hipStreamCaptureStatusNone && dbuf_reserve(c, c->part, I8_PART_BYTES, false)) return bgl_last_code();
    if (ks <= 1) return 0;
    const size_t need = i8_part(L, ks) + (L.xf ? L.M * 4 : 0);
    if (need > I8_PART_BYTES || (c->fixed_base && c->fixed_used + need + 256 > c->fixed_cap)) return 0;
    if (dbuf_reserve(c, c->part, c->fixed_base ? need : I8_PART_BYTES, false)) return bgl_last_code();
    int *p = (int *)c->part.p;
    for (int i = 0; i < L.n; i++) {
        L.t[i].part = p;
        p += (size_t)ks * L.M * ((L.t[i].T.N + 3) & ~3);
    }
    if (L.xf) L.xs = L.xs_out = (float *)p;
    L.ks = ks;
    return 0;
}

// Columns whose codes each workgroup of k_i8_s makes itself, where it has registers for all values: it costs less than the
// launch that quantizes them up to 8192 values, and in one column, which that launch gives to one CU, up to 16384.  us with
// this / with the launch (columns x channels x K): 1 x 4096 x 4096 6.2 / 8.2, 1 x 14336 x 4096 14.0 / 16.6, 1 x 4096 x 14336
// 16.3 / 17.2, 2 x 4096 x 4096 7.1 / 8.4, 4 x 4096 x 4096 8.9 / 8.6, 16 x 8960 x 1024 8.8 / 8.3.
static bool f32_fits(int M, int K, int units, int ks) {
    return M <= 16 && K % 64 == 0 && M * (long)K <= (M == 1 ? 16384 : 8192) && M * (long)(K / 64) <= 4l * I8_S_RND * std::min(16, std::max(1, units / ks));
}

template <int RB, int CB, bool GLU>
static void s_go(const I8Launch &L, int blocks, hipStream_t st) {
    constexpr int D = RB + CB <= 2 ? 4 : 2;
    const int nw = std::min(i8_s_waves<RB, CB>(), std::max(1, L.t[0].T.nunits / L.ks));
    const size_t lds = (size_t)std::min(nw * RB * CB, I8_S_PART) * 1024;
    const dim3 grid(blocks, (L.M + 63) / 64, L.ks);
    if constexpr (CB == 1)
        if (L.xf) {
            hipLaunchKernelGGL((k_i8_s<RB, 1, D, true, GLU>), grid, dim3(nw * 64), lds + (size_t)L.M * (L.t[0].T.K + 16) + L.M * 4, st, L);
            return;
        }
    hipLaunchKernelGGL((k_i8_s<RB, CB, D, false, GLU>), grid, dim3(nw * 64), lds, st, L);
}
// workgroups of RB blocks of 16 channels; of a pair, half of them gate's
static long s_blocks(I8Launch &L, int RB) {
    if (L.glu) return ((L.t[0].T.N + 15) / 16 + RB / 2 - 1) / (RB / 2);
    long blocks = 0;
    for (int i = 0; i < L.n; i++) {
        L.t[i].blk0 = (int)blocks;
        blocks += ((L.t[i].T.N + 15) / 16 + RB - 1) / RB;
    }
    return blocks;
}
static int run_s(bgl_ctx *c, I8Launch &L, int RB, int ks) {
    const int rc = L.glu ? 0 : i8_split(c, L, ks), CB = std::min(4, (L.M + 15) / 16);
    if (rc) return rc;
    if (L.glu) L.ks = 1;
    const int blocks = (int)s_blocks(L, RB);
#define GO(R, C) if (RB == R && CB == C) s_go<R, C, true>(L, blocks, c->stream)
    if (L.glu) {
        GO(2, 1); GO(2, 2); GO(2, 3); GO(2, 4); GO(4, 1); GO(4, 2); GO(4, 3); GO(4, 4);
        return 0;
    }
#undef GO
#define GO(R, C) if (RB == R && CB == C) s_go<R, C, false>(L, blocks, c->stream)
    GO(1, 1); GO(1, 2); GO(1, 3); GO(1, 4); GO(2, 1); GO(2, 2); GO(2, 3); GO(2, 4); GO(4, 1); GO(4, 2); GO(4, 3); GO(4, 4);
#undef GO
    return 0;
}

static long l_tiles(I8Launch &L, int BM, int BN) {
    long ntn = 0;
    for (int i = 0; i < L.n; i++) {
        L.t[i].blk0 = (int)ntn;
        ntn += (L.t[i].T.N + BN - 1) / BN;
    }
    return ntn * ((L.M + BM - 1) / BM);
}
template <int CM, int CN, int NWM, int NWN>
static int run_l(bgl_ctx *c, I8Launch &L, int ks) {
    constexpr int BM = 16 * CM * NWM, BN = 16 * CN * NWN;
    const int rc = i8_split(c, L, ks);
    if (rc) return rc;
    const int ntm = (L.M + BM - 1) / BM, ntn = (int)(l_tiles(L, BM, BN) / ntm);
    const size_t lds = 2 * (size_t)(BM + BN) * 128;
    auto kern = k_i8_l<CM, CN, NWM, NWN>;
    HIPCHK(hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    hipLaunchKernelGGL(kern, dim3((unsigned)ntm * ntn, 1, L.ks), dim3(NWM * NWN * 64), lds, c->stream, L, ntm, ntn);
    return 0;
}

// Which kernel runs a product of M columns, by the time in us that each would take: the launch and the sums of a tile
// (constant), what a CU reads or multiplies for its tiles, and with K split the launch that joins the slices.  The
// constants were fitted to 37 shapes from 1 x 256 x 1536 to 4096 x 14336 x 4096, where the choice is the fastest of all
// or within a tenth; us of both sides of each line (columns x channels x K):
//   up to 64 columns, k_i8_s with 16 / 32 / 64 channels a workgroup: 1 x 4096 x 4096 5.5 / 5.8 / 6.4, 1 x 8960 x 1536
//     8.0 / 6.5 / 5.5, 64 x 14336 x 4096 40.8 / 26.6 / 21.0; 64 with K in 1 / 4 / 8 slices: 64 x 1536 x 8960
//     24.8 / 13.1 / 12.1, 64 x 14336 x 4096 21.5 / 34.0 / 51.7
//   k_i8_s with 64 x 64 outputs / 128 x 128 tiles / 256 x 256: 512 x 1536 x 1536 9.3 / 12.8 / 31.8, 2048 x 2048 x 2048
//     34.8 / 16.4 / 33.3, 2048 x 14336 x 4096 369 / 153 / 126
//   128 x 192 tiles / 128 x 128, where the last round of the latter leaves most CUs idle: 512 x 17920 x 1536 24.6 / 29.4,
//     1500 x 6144 x 4096 45.5 / 59.0, 2048 x 8960 x 1536 38.1 / 44.6; where it does not: 512 x 14336 x 4096 50.8 / 41.7.
//     Up to 512 tiles of 128 x 192 (80 KB of LDS, 114 registers) are all there at once, two on a CU, and a step of K takes
//     1.3 to 1.8 us for both; more follow one another at 0.8 to 1.0 a round.  us a step at K = 4096 by rounds of 256 tiles:
//     0.5 0.73, 1 1.02, 1.2 1.4, 1.5 1.3 to 1.5, 2 1.8, 2.5 2.7, 3 2.8 to 2.9, 4 3.6, 6 5.2, 9 7.6, 12 10.3.  Over 36 shapes of
//     512 and 1500 columns, 6144 to 49152 channels, K of 1536 and 4096 the choice is the fastest of the three tiles each time
//   128 x 128 tiles with K in 1 / 4 slices: 1024 x 1536 x 8960 48.7 / 31.1, 128 x 8960 x 1536 14.0 / 19.9
static int run_any(bgl_ctx *c, I8Launch &L) {
    const int K = L.t[0].T.K, M = L.M;
    auto up = [](long v) { return (double)((v + I8_CUS - 1) / I8_CUS); };
    auto join = [&](int ks) { return ks > 1 ? 3.0 + i8_part(L, ks) / I8_JOIN : 0.0; };
    if (M <= 64) {
        int best = 0, bks = 1;
        double least = 1e30;
        for (int RB = L.glu ? 2 : 1; RB <= 4; RB *= 2) {
            const long blocks = s_blocks(L, RB);
            for (int ks = 1; ks <= 8 && (ks == 1 || (!L.glu && K / ks >= I8_SLICE)); ks *= 2) {
                if (L.xf && !f32_fits(M, K, L.t[0].T.nunits, ks)) break;
                const double us = up(blocks * ks) * ((double)(16 * RB + M) * K / ks / 40e3 + 1.5) + join(ks);
                if (us < least) { least = us; best = RB; bks = ks; }
            }
        }
        return run_s(c, L, best, bks);
    }
    const double ns = (K + 127) / 128;
    const long t256 = l_tiles(L, 256, 256), t128 = l_tiles(L, 128, 128), t64 = s_blocks(L, 4) * ((M + 63) / 64);
    int ks = 1;
    double c128 = 1e30;
    for (int k = 1; k <= 8 && (k == 1 || (t128 < I8_CUS && K / k >= I8_SLICE)); k *= 2) {
        const double r = (double)t128 * k / I8_CUS;
        const double us = 4.0 + (r <= 1.0 ? 0.62 + 0.25 * r : 0.6 * up(t128 * k)) * ns / k + join(k);
        if (us < c128) { c128 = us; ks = k; }
    }
    const double c256 = 6.0 + 1.9 * ns * up(t256);
    const double c64 = 3.0 + (t64 <= I8_CUS ? 0.4 : 0.62 * up(t64)) * ns;
    const double u192 = up(l_tiles(L, 128, 192));
    const double c192 = 6.0 + (u192 == 2.0 ? 1.44 : 0.85 * u192) * ns;      // 2: both tiles of a CU at once
    if (c64 <= c128 && c64 <= c192 && c64 <= c256 && (M + 63) / 64 <= 65535) return run_s(c, L, 4, 1);
    if (c192 < c128 && c192 <= c256) return run_l<4, 3, 2, 4>(c, L, 1);
    if (c128 <= c256) return run_l<4, 2, 2, 4>(c, L, ks);
    return run_l<8, 4, 2, 4>(c, L, 1);
}

int run_i8(bgl_ctx *c, int n, const BglDevTensor *Ts, const int8_t *xq, long ldq, const float *xs, const float *const *bias,
           void *const *y, int y_type, const long *ldy, int M, const float *xf, bool glu) {
    I8Launch L;
    memset(&L, 0, sizeof L);
    L.n = n; L.M = M; L.glu = glu; L.K16 = (Ts[0].K + 15) & ~15; L.y_type = y_type;
    L.xq = xq; L.ldq = ldq; L.xs = xs; L.xf = xf;
    int widest = 0;
    for (int i = 0; i < n; i++) {
        I8Task &t = L.t[i];
        t.T = Ts[i];
        t.bias = bias ? bias[i] : nullptr;
        t.y = y[i];
        t.ldy = ldy ? ldy[i] : Ts[i].N;
        widest = std::max(widest, Ts[i].N);
    }
    int tok = prof_begin(c, 1);
    const int rc = run_any(c, L);
    if (!rc && L.ks > 1) {
        for (int i = 0; i < n; i++) L.t[i].blk0 = i;
        hipLaunchKernelGGL(k_i8_join, dim3((unsigned)((widest + 1023) / 1024), M, n), dim3(256), 0, c->stream, L);
    }
    prof_end(c, tok);
    if (rc) return rc;
    HIPCHK(hipGetLastError());
    return 0;
}

int prep_i8_cols(bgl_ctx *c, const float *x, const float *u, float *h, int M, int K, bool reuse) {
    const long ldq = i8_ld_scratch(K);
    if (dbuf_reserve(c, c->act_w, (size_t)M * ldq, false) || dbuf_reserve(c, c->act_s, (size_t)M * 4, false)) return bgl_last_code();
    c->prep_reuse = false;
    int rc = run_quant_rows(c, x, u, h, M, K, (int8_t *)c->act_w.p, ldq, (float *)c->act_s.p);
    if (rc) return rc;
    c->prep_act = BGL_ACT_W4A8; c->prep_gq = PREP_GQ_TOKEN; c->prep_M = M; c->prep_K = K; c->prep_x = nullptr;
    c->prep_reuse = reuse;
    return 0;
}

int run_i8_cols(bgl_ctx *c, int n, const BglDevTensor *Ts, const float *x, const float *u, float *h, int M,
                const float *const *bias, float *const *y, bool glu) {
    void *yv[BGL_MAX_TASKS];
    for (int i = 0; i < n; i++) yv[i] = y[glu ? 0 : i];
    if (!u && f32_fits(M, Ts[0].K, Ts[0].nunits, 1) && (uintptr_t)x % 16 == 0)
        return run_i8(c, n, Ts, nullptr, 0, nullptr, bias, yv, BGL_T_F32, nullptr, M, x, glu);
    int rc = prep_i8_cols(c, x, u, h, M, Ts[0].K, false);
    if (rc) return rc;
    return run_i8(c, n, Ts, (const int8_t *)c->act_w.p, i8_ld_scratch(Ts[0].K), (const float *)c->act_s.p, bias, yv, BGL_T_F32,
                  nullptr, M, nullptr, glu);
}

extern "C" int bgl_matmul_i8_dev(bgl_ctx *c, int n, const bgl_tensor *const *w, const int8_t *xq, long ldq, const float *xs,
                                 const float *const *bias, void *const *y, int y_type, const long *ldy, int M) {
    if (!c || n < 1 || n > BGL_MAX_TASKS || !w || !xq || !xs || !y || M < 1)
        return bgl_fail(BGL_E_ARG, "bgl_matmul_i8_dev: bad argument");
    if (y_type != BGL_T_F32 && y_type != BGL_T_F16 && y_type != BGL_T_BF16)
        return bgl_fail(BGL_E_ARG, "bgl_matmul_i8_dev: unknown element type %d", y_type);
    BglDevTensor Ts[BGL_MAX_TASKS];
    for (int i = 0; i < n; i++) {
        if (!w[i] || !w[i]->experts.empty() || !y[i]) return bgl_fail(BGL_E_ARG, "bgl_matmul_i8_dev: tensor %d invalid", i);
        Ts[i] = w[i]->T;
        if (Ts[i].fmt != BGL_K_Q8C) return bgl_fail(BGL_E_UNSUPPORTED, "bgl_matmul_i8_dev: kind %d is not K_Q8C", Ts[i].fmt);
        if (Ts[i].K != Ts[0].K) return bgl_fail(BGL_E_ARG, "bgl_matmul_i8_dev: fused tensors must share in");
        if (ldy && ldy[i] < Ts[i].N) return bgl_fail(BGL_E_ARG, "bgl_matmul_i8_dev: y rows %ld apart, %d values each", ldy[i], Ts[i].N);
    }
    if (ldq < Ts[0].K || ldq % 16 || (uintptr_t)xq % 16)
        return bgl_fail(BGL_E_ARG, "bgl_matmul_i8_dev: code rows are 16-byte aligned, a multiple of 16 and at least in=%d bytes apart (ldq=%ld)",
                        Ts[0].K, ldq);
    if (ldq > (1l << 22)) return bgl_fail(BGL_E_ARG, "bgl_matmul_i8_dev: code rows %ld bytes apart (at most %ld)", ldq, 1l << 22);
    HIPCHK(hipSetDevice(c->device));
    return run_i8(c, n, Ts, xq, ldq, xs, bias, y, y_type, ldy, M);
}
