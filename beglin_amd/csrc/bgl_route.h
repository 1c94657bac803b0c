// bgl_route.h -- one token's routing on the device: an expert's score by one wave, and the softmax, top-K and
// renorm of a token's scores by one wave (moe_ffn_batched's routing, qwen_infer.c:5243-5257, :5275).
#pragma once
#include "bgl_internal.h"

#define ROUTE_MAXE 256
#define ROUTE_RND 8

// The wave's dot product of a router row and a token row in double; valid in every lane.  Each lane sums its elements
// 4*lane + 256*i in ascending order; a round's 8 row and 8 x loads all go out before the first fma
// (buffer loads: the ones past H return zero, so none is conditional and one round trip serves
// H <= 2048).
__device__ __forceinline__ double route_dot_wave(const float *w, const float *x, int H, int lane) {
    const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(w), (short)0, H * 4, 0x00020000);
    const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(x), (short)0, H * 4, 0x00020000);
    typedef float rf4 __attribute__((ext_vector_type(4)));
    double acc = 0.0;
    for (int c0 = 0; c0 < H; c0 += ROUTE_RND * 256) {
        rf4 wv[ROUTE_RND], xv[ROUTE_RND];
#pragma unroll
        for (int i = 0; i < ROUTE_RND; i++) {
            const int off = (c0 + 256 * i + 4 * lane) * 4;
            wv[i] = __builtin_bit_cast(rf4, __builtin_amdgcn_raw_buffer_load_b128(wr, off, 0, 0));
            xv[i] = __builtin_bit_cast(rf4, __builtin_amdgcn_raw_buffer_load_b128(xr, off, 0, 0));
        }
#pragma unroll
        for (int i = 0; i < ROUTE_RND; i++) {
            acc = fma((double)wv[i].x, (double)xv[i].x, acc);
            acc = fma((double)wv[i].y, (double)xv[i].y, acc);
            acc = fma((double)wv[i].z, (double)xv[i].z, acc);
            acc = fma((double)wv[i].w, (double)xv[i].w, acc);
        }
    }
    for (int o = 32; o; o >>= 1) acc += __shfl_xor(acc, o);
    return acc;
}

// Softmax, top-K and renorm of one token's E scores by one wave; lane k < K returns pick k.
__device__ __forceinline__ void route_topk_wave(const float *__restrict__ sc_t, int E, int K, int renorm, int lane,
                                                int &sel_i, float &sel_w, float *lbuf) {
    constexpr int PL = ROUTE_MAXE / 64;                      // scores per lane: expert lane + 64j
    float v[PL];
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < PL; j++) {
        const int e = lane + 64 * j;
        v[j] = e < E ? sc_t[e] : 0.0f;
        if (e < E) mx = fmaxf(mx, v[j]);
    }
    mx = wave_max_f32(mx);
#pragma unroll
    for (int j = 0; j < PL; j++) {
        const int e = lane + 64 * j;
        if (e < E) v[j] = (float)exp((double)__fsub_rn(v[j], mx));
    }
    // the double sum in expert order: the values go through the wave's LDS row (lbuf, 16-byte
    // aligned, ROUTE_MAXE floats) and every lane reads them all at the same addresses (broadcast
    // reads, 16 values per round); a wave's LDS accesses complete in order
#pragma unroll
    for (int j = 0; j < PL; j++)
        if (lane + 64 * j < E) lbuf[lane + 64 * j] = v[j];
    __builtin_amdgcn_wave_barrier();
    typedef float lf4 __attribute__((ext_vector_type(4)));
    const lf4 *l4 = reinterpret_cast<const lf4 *>(lbuf);
    double sum = 0.0;
    int e16 = 0;
    for (; e16 + 16 <= E; e16 += 16) {
        const lf4 q0 = l4[e16 / 4], q1 = l4[e16 / 4 + 1], q2 = l4[e16 / 4 + 2], q3 = l4[e16 / 4 + 3];
        sum += (double)q0.x; sum += (double)q0.y; sum += (double)q0.z; sum += (double)q0.w;
        sum += (double)q1.x; sum += (double)q1.y; sum += (double)q1.z; sum += (double)q1.w;
        sum += (double)q2.x; sum += (double)q2.y; sum += (double)q2.z; sum += (double)q2.w;
        sum += (double)q3.x; sum += (double)q3.y; sum += (double)q3.z; sum += (double)q3.w;
    }
    for (; e16 < E; e16++) sum += (double)lbuf[e16];
    sel_i = 0;
    sel_w = 0.0f;
#pragma unroll
    for (int j = 0; j < PL; j++) {
        if (64 * j < E) v[j] = (float)((double)v[j] / sum);
        if (!(lane + 64 * j < E && v[j] >= 0.0f)) v[j] = -1.0f;     // not there, or NaN: never picked
    }
    for (int k = 0; k < K; k++) {
        // the wave's largest value left, of the lowest expert that has it; none left: -1 and no expert
        float bv = v[0];
#pragma unroll
        for (int j = 1; j < PL; j++) bv = fmaxf(bv, v[j]);
        bv = wave_max_f32(bv);
        int bi = 0x7fffffff;
#pragma unroll
        for (int j = PL - 1; j >= 0; j--) {
            const uint64_t m = __builtin_amdgcn_ballot_w64(v[j] == bv);
            if (m != 0 && bv >= 0.0f) bi = 64 * j + __builtin_ctzll(m);
        }
#pragma unroll
        for (int j = 0; j < PL; j++)
            if (lane + 64 * j == bi) v[j] = -1.0f;
        if (lane == k) { sel_w = bv; sel_i = bi; }
    }
    if (renorm) {
        double s = 0.0;
        for (int k = 0; k < K; k++) s += (double)rlane_f(sel_w, k);
        if (s > 0.0) sel_w = (float)((double)sel_w / s);
    }
}
