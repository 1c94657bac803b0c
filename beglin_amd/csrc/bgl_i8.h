// bgl_i8.h -- what the kernels of the int8 scheme share (codes with one scale per token and per output
// channel): element types in memory, the per-token quantizer, and the matrix-core operands.
#pragma once
#include "bgl_internal.h"

#define I8_MAX_K 131071          // |code| <= 128: the int32 sum of this many products stays below 2^31
typedef int i8_i4 __attribute__((ext_vector_type(4)));
typedef unsigned int i8_u4 __attribute__((ext_vector_type(4)));
typedef float i8_f4 __attribute__((ext_vector_type(4)));

static inline size_t i8_elem(int type) { return type == BGL_T_F32 ? 4 : 2; }

// ------------------------------------------------------------------ element types
// One value of a row in fp32, fp16 or bf16 (every one of them is an fp32 value exactly).  fp16 is read as the integer that
// i8_st stores: a thread may read back what it wrote, and accesses of two types may change places.
__device__ __forceinline__ float i8_ld(const void *p, int type, size_t i) {
    if (type == BGL_T_F32) return ((const float *)p)[i];
    if (type == BGL_T_F16) return (float)__builtin_bit_cast(_Float16, ((const uint16_t *)p)[i]);
    return __uint_as_float((uint32_t)((const uint16_t *)p)[i] << 16);
}
// fp32 to the type, to nearest, ties to even; the bf16 cast keeps NaN a NaN.
__device__ __forceinline__ uint16_t i8_h16(float v, int type) {
    if (type == BGL_T_F16) return __builtin_bit_cast(uint16_t, (_Float16)v);
    return __builtin_bit_cast(uint16_t, (__bf16)v);
}
__device__ __forceinline__ void i8_st(void *p, int type, size_t i, float v) {
    if (type == BGL_T_F32) ((float *)p)[i] = v;
    else ((uint16_t *)p)[i] = i8_h16(v, type);
}
// the fp32 value that a store in this type keeps
__device__ __forceinline__ float i8_kept(float v, int type) {
    if (type == BGL_T_F32) return v;
    const uint16_t h = i8_h16(v, type);
    return type == BGL_T_F16 ? (float)__builtin_bit_cast(_Float16, h) : __uint_as_float((uint32_t)h << 16);
}

// ------------------------------------------------------------------ the per-token quantizer
// q4_quant_act_i8's arithmetic (q4gemv.h:177-213) with the whole row as the group: mx = max(1e-8, max|x|),
// sc = mx / 127, inv = 1 / sc, code = sat8(trunc(x * inv +- 0.5)).  The maximum is taken on the bits of
// |x|, where NaN lies above Inf: a row holding either gets the scale NaN or Inf and every code 0, so its
// products are NaN.
#define I8_MX0 0x322BCC77u       // 1e-8f
struct I8Scale {
    float sc, inv;
    bool nf;
};
__device__ __forceinline__ I8Scale i8_scale(uint32_t mxbits) {
    I8Scale s;
    s.nf = mxbits >= 0x7f800000u;
    s.sc = __fdiv_rn(__uint_as_float(mxbits), 127.0f);
    s.inv = __fdiv_rn(1.0f, s.sc);
    return s;
}
__device__ __forceinline__ int i8_code(float v, const I8Scale &s) {
    const float p = s.nf ? 0.0f : __fmul_rn(v, s.inv);        // |p| <= 127 and a rounding
    const int q = (int)__fadd_rn(p, p >= 0.0f ? 0.5f : -0.5f);
    return q > 127 ? 127 : (q < -128 ? -128 : q);
}
__device__ __forceinline__ uint32_t i8_pack4(int a, int b, int c, int d) {
    return (uint32_t)(a & 255) | ((uint32_t)(b & 255) << 8) | ((uint32_t)(c & 255) << 16) | ((uint32_t)d << 24);
}

// k_swiglu's arithmetic (bgl_mlp.hip): g / (1 + exp(-g)) * u, the exponential rounded once from double
__device__ __forceinline__ float i8_swiglu(float g, float u) {
    const float e = (float)exp(-(double)g);
    return __fmul_rn(__fdiv_rn(g, __fadd_rn(1.0f, e)), u);
}

// the output of a product: the int32 sum, rounded once to fp32 (it can pass 2^24), times the rounded
// product of its two scales
__device__ __forceinline__ float i8_out(int acc, float as, float ws) { return __fmul_rn((float)acc, __fmul_rn(as, ws)); }

// ------------------------------------------------------------------ host side
// M fp32 rows to codes [M][ldq] (bytes K .. ldq zeroed) and scales [M]; u != null: the rows are h = silu(x) * u,
// also written to h.  (bgl_norm.hip)
int run_quant_rows(bgl_ctx *c, const float *x, const float *u, float *h, int M, int K, int8_t *xq, long ldq, float *xs);
// n <= 4 tensors of the int8 kind over M columns of codes (bgl_i8.hip); y[i] rows ldy[i] values apart.  xf: fp32 columns in
// place of the codes (run_i8_cols)
int run_i8(bgl_ctx *c, int n, const BglDevTensor *Ts, const int8_t *xq, long ldq, const float *xs, const float *const *bias,
           void *const *y, int y_type, const long *ldy, int M, const float *xf = nullptr, bool glu = false);
// M fp32 columns (u, h as run_quant_rows) quantized into the context's act_w / act_s; reuse: for
// bgl_matmul_prepped_dev, as columns with one scale per token
#define PREP_GQ_TOKEN -1
int prep_i8_cols(bgl_ctx *c, const float *x, const float *u, float *h, int M, int K, bool reuse);
// run_i8 over fp32 columns, quantized first; glu (M <= 64): Ts are gate and up of one h = silu(gate x) * up x, written to
// y[0]
int run_i8_cols(bgl_ctx *c, int n, const BglDevTensor *Ts, const float *x, const float *u, float *h, int M,
                const float *const *bias, float *const *y, bool glu = false);
// bytes between the codes' rows in the context's scratch: whole 64-value units
static inline long i8_ld_scratch(int K) { return ((long)K + 63) / 64 * 64; }
// The routed FFN of K_Q8C experts (bgl_moe_i8.hip), shapes checked by the caller: routing given (rw null), or from the
// router rw [E][H] (+ rb).
#define MOE_I8_MAX_E 1024
int run_moe_i8(bgl_ctx *c, const bgl_tensor *gate, const bgl_tensor *up, const bgl_tensor *down, const bgl_tensor *sg, const bgl_tensor *su,
               const bgl_tensor *sd, const float *rw, const float *rb, int renorm, const float *x, const int32_t *idx, const float *w, int T,
               int K, float *out);
