// bgl_kv.h -- the paged cache of keys and values in 4 bits: where a record keeps what (16 tokens of one head, K before V;
// include/beglin_qgemv.h has the layout), and the checks of its descriptor.
//
// The record is laid out for the matrix cores, which want the values that a product sums side by side in a lane:
// v_mfma_f32_16x16x32_f16 takes 8 of them from lane l, for row or column l % 16 and the (l / 16)-th eighth of the sum.
//   scores  sum over a head's values: lane (b = l / 16, token = l % 16) owns values 8 G b .. 8 G b + 8 G - 1 of its token, 4 G
//           bytes in one piece, and all lanes together read 64 pieces in a row.  A dword's nibbles are placed so that
//           (w >> 0 or 8) & 0x000f000f and & 0x00f000f0 are pairs of neighbours.
//   output  sum over tokens: lane (b, n = l % 16) owns values 2 G n .. 2 G n + 2 G - 1 of tokens 4 b .. 4 b + 3, again 4 G
//           bytes in one piece.  A dword holds two values of four tokens, so the same masks give pairs of tokens
//           (0, 2) and (1, 3) of one value: no transposition anywhere.
// An fp16 with exponent 2^10 (or 2^6) and a code in its lowest (or fourth to seventh) mantissa bits is 1024 + c (64 + c), so a
// pair of codes becomes a pair of values by and/or, a subtraction, which is exact, and one multiply-add: the definition's
// single rounding.
#pragma once
#include "bgl_i8.h"

typedef _Float16 kv_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 kv_h8 __attribute__((ext_vector_type(8)));
typedef float kv_f4 __attribute__((ext_vector_type(4)));

#define KV_TILE 16
static inline bool kv_dim_ok(int D) { return D == 64 || D == 96 || D == 128 || D == 192 || D == 256; }

// byte offsets inside a record of 20 D bytes
__host__ __device__ __forceinline__ int kv_record(int D) { return 20 * D; }
__host__ __device__ __forceinline__ int kv_k_steps(int D) { return 8 * D; }
__host__ __device__ __forceinline__ int kv_v_codes(int D) { return 10 * D; }
__host__ __device__ __forceinline__ int kv_v_steps(int D) { return 18 * D; }

// The record of a slot and head; the slot lies in the cache.
__device__ __forceinline__ uint8_t *kv_at(const bgl_kv &c, int slot, int head) {
    const int pg = slot / c.page, in = slot - pg * c.page;
    return (uint8_t *)c.data + (((size_t)pg * c.heads + head) * (c.page / KV_TILE) + in / KV_TILE) * kv_record(c.D);
}

// 8 values anywhere in memory (gfx950 loads and stores 16 bytes at any address)
typedef float kv_mf4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned int kv_mu4 __attribute__((ext_vector_type(4), aligned(2)));

__device__ __forceinline__ void kv_load8(float (&q)[8], const void *p, int type, long at) {
    if (type == BGL_T_F32) {
        const kv_mf4 *s = (const kv_mf4 *)((const float *)p + at);
        const kv_mf4 u = s[0], v = s[1];
#pragma unroll
        for (int j = 0; j < 4; j++) { q[j] = u[j]; q[4 + j] = v[j]; }
        return;
    }
    const kv_mu4 u = *(const kv_mu4 *)((const uint16_t *)p + at);
    if (type == BGL_T_F16) {
#pragma unroll
        for (int j = 0; j < 8; j++) q[j] = (float)__builtin_bit_cast(_Float16, (uint16_t)(u[j / 2] >> (16 * (j & 1))));
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) q[j] = __uint_as_float(j & 1 ? u[j / 2] & 0xffff0000u : u[j / 2] << 16);
    }
}
__device__ __forceinline__ void kv_store8(void *p, int type, long at, const float (&q)[8]) {
    if (type == BGL_T_F32) {
        kv_mf4 *s = (kv_mf4 *)((float *)p + at);
        s[0] = kv_mf4{q[0], q[1], q[2], q[3]};
        s[1] = kv_mf4{q[4], q[5], q[6], q[7]};
        return;
    }
    kv_mu4 u;
    if (type == BGL_T_F16) {
#pragma unroll
        for (int j = 0; j < 4; j++) u[j] = __builtin_bit_cast(uint32_t, kv_h2{(_Float16)q[2 * j], (_Float16)q[2 * j + 1]});
    } else {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int j = 0; j < 4; j++) u[j] = __builtin_bit_cast(uint32_t, b2{(__bf16)q[2 * j], (__bf16)q[2 * j + 1]});
    }
    *(kv_mu4 *)((uint16_t *)p + at) = u;
}

// 4 values
__device__ __forceinline__ void kv_store4(void *p, int type, long at, kv_f4 q) {
    typedef unsigned int u2 __attribute__((ext_vector_type(2), aligned(2)));
    if (type == BGL_T_F32) *(kv_mf4 *)((float *)p + at) = q;
    else *(u2 *)((uint16_t *)p + at) = u2{(uint32_t)i8_h16(q[0], type) | (uint32_t)i8_h16(q[1], type) << 16,
                                          (uint32_t)i8_h16(q[2], type) | (uint32_t)i8_h16(q[3], type) << 16};
}
// The descriptor's checks (bgl_heads.hip); 0 or an error code.
int kv_check(const char *who, const bgl_kv *kv);
// Rows [n][heads][D] at a pointer: tokens ld apart and heads hd, both at least one row of what they step over, in either order.
bool kv_rows_ok(long ld, long hd, long n, long heads, long D);
