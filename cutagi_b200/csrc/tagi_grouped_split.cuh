// Pieces shared by the tensor-core kernels of the Linear layers grouped by expert (tagi_grouped_tc.cu,
// tagi_grouped_thin.cu): the exact split of floats into bf16 parts and the products of the parts.
#pragma once
#include "tagi_grouped.h"
#include "tagi_tc_ptx.cuh"

namespace tagi {
namespace {

using namespace ptx;

__device__ __forceinline__ int round_up(int a, int b) { return (a + b - 1) / b * b; }

// Four floats, STRIDE apart, of which those at offsets below `valid` exist; the others are zero. VEC (STRIDE 1): all four or
// none, 16-byte aligned.
template <bool VEC, int STRIDE = 1>
__device__ __forceinline__ float4 ld4(const float *p, int valid) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (VEC) {
        if (valid > 0) v = __ldg(reinterpret_cast<const float4 *>(p));
    } else {
        if (valid > 0) v.x = __ldg(p);
        if (valid > STRIDE) v.y = __ldg(p + STRIDE);
        if (valid > 2 * STRIDE) v.z = __ldg(p + 2 * STRIDE);
        if (valid > 3 * STRIDE) v.w = __ldg(p + 3 * STRIDE);
    }
    return v;
}

// Four bytes to shared memory, or to global memory, if i < n: one instruction each, no branch. With branches around them the
// columns of a tile's output take turns waiting (parameter pass, 100 rows of each of 8 experts of 4096 x 4096: 971 us, so 639 us).
__device__ __forceinline__ void copy_below(uint32_t dst, const float *src, int i, int n) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.s32 p, %2, %3;\n\t@p cp.async.ca.shared.global [%0], [%1], 4;\n\t}" ::"r"(dst), "l"(src), "r"(i), "r"(n) : "memory");
}
__device__ __forceinline__ void store_below(float *dst, float v, int i, int n) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.s32 p, %2, %3;\n\t@p st.global.f32 [%0], %1;\n\t}" ::"l"(dst), "f"(v), "r"(i), "r"(n) : "memory");
}

// Which of 16 contraction steps lies at place j of an operand whose steps run along memory. SPREAD: rows that are not aligned
// to 16 bytes are read a float at a time; four lanes then take neighbouring steps (half the sectors of taking every fourth),
// which leaves a lane with steps 4 apart in four neighbouring places. The order of the steps does not matter to a sum as
// long as both operands have the same.
template <bool SPREAD>
__device__ __forceinline__ int step_at(int j) {
    return SPREAD ? (j & ~15) | ((j & 3) << 2) | ((j >> 2) & 3) : j;
}

__device__ __forceinline__ uint32_t top_halves(float a, float b) {   // a's upper 16 bits below b's
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, 0x7632;" : "=r"(r) : "r"(__float_as_uint(a)), "r"(__float_as_uint(b)));
    return r;
}
__device__ __forceinline__ float truncated(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
// two 32-bit operations as one instruction
__device__ __forceinline__ void add2(float &a, float &b, float x, float y) {
    asm("{\n\t.reg .b64 s, t;\n\tmov.b64 s, {%0, %1};\n\tmov.b64 t, {%2, %3};\n\tadd.rn.f32x2 s, s, t;\n\tmov.b64 {%0, %1}, s;\n\t}"
        : "+f"(a), "+f"(b)
        : "f"(x), "f"(y));
}
__device__ __forceinline__ void subtract_truncated2(float &a, float &b) {
    const float x = truncated(a), y = truncated(b);
    asm("{\n\t.reg .b64 s, t;\n\tmov.b64 s, {%0, %1};\n\tmov.b64 t, {%2, %3};\n\tsub.rn.f32x2 s, s, t;\n\tmov.b64 {%0, %1}, s;\n\t}"
        : "+f"(a), "+f"(b)
        : "f"(x), "f"(y));
}
__device__ __forceinline__ void sts64(uint32_t at, uint32_t a, uint32_t b) {
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(a), "r"(b) : "memory");
}
// hi, mid, lo of four values to their part tiles, `part` bytes apart
__device__ __forceinline__ void store_split(uint32_t at, uint32_t part, float4 v) {
    sts64(at, top_halves(v.x, v.y), top_halves(v.z, v.w));
    subtract_truncated2(v.x, v.y), subtract_truncated2(v.z, v.w);
    sts64(at + part, top_halves(v.x, v.y), top_halves(v.z, v.w));
    subtract_truncated2(v.x, v.y), subtract_truncated2(v.z, v.w);
    sts64(at + 2 * part, top_halves(v.x, v.y), top_halves(v.z, v.w));
}
__device__ __forceinline__ float4 squared(float4 v) { return make_float4(v.x * v.x, v.y * v.y, v.z * v.z, v.w * v.w); }

// kind::f16 instruction descriptor: FP32 accumulation, bf16 operands (see make_idesc_tf32 for the fields)
__host__ __device__ constexpr uint32_t make_idesc_bf16(int M, int N, int a_mn, int b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}
// The six products of 16 contraction steps. The parts of A lie AP units of 16 bytes apart, those of B BP; the high descriptor
// words are the same for all. One asm block each: building descriptors between the instructions costs the issuing thread
// more than the tensor core needs for a narrow tile.
#define GROUPED_MMA(CG, XA, XB, P)                                                    \
    "add.u32 ra, %1, " XA ";\n\tadd.u32 rb, %2, " XB ";\n\t"                          \
    "mov.b64 da, {ra, %3};\n\tmov.b64 db, {rb, %3};\n\t"                              \
    "tcgen05.mma.cta_group::" CG ".kind::f16 [%0], da, db, %4, " P ";\n\t"
// lo hi, hi lo, mid mid, mid hi, hi mid; accumulate == 0: the first overwrites the accumulator
#define GROUPED_SMALL(CG)                                                                                          \
    asm volatile(                                                                                                  \
        "{\n\t.reg .pred p, t;\n\t.reg .b32 ra, rb;\n\t.reg .b64 da, db;\n\t"                                    \
        "setp.ne.b32 p, %5, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"                                                       \
        GROUPED_MMA(CG, "%8", "0", "p") GROUPED_MMA(CG, "0", "%9", "t") GROUPED_MMA(CG, "%6", "%7", "t")           \
        GROUPED_MMA(CG, "%6", "0", "t") GROUPED_MMA(CG, "0", "%7", "t") "}"                                        \
        ::"r"(d), "r"(x), "r"(y), "r"(hi), "r"(idesc), "r"(accumulate), "n"(AP), "n"(BP), "n"(2 * AP), "n"(2 * BP) \
        : "memory")
#define GROUPED_LARGE(CG)                                                                                          \
    asm volatile(                                                                                                  \
        "{\n\t.reg .pred t;\n\t.reg .b32 ra, rb;\n\t.reg .b64 da, db;\n\tsetp.eq.b32 t, 0, 0;\n\t"                \
        GROUPED_MMA(CG, "0", "0", "t") "}"                                                                         \
        ::"r"(d), "r"(x), "r"(y), "r"(hi), "r"(idesc)                                                              \
        : "memory")
template <uint32_t AP, uint32_t BP>
__device__ __forceinline__ void mma_small_products(uint32_t d, uint32_t x, uint32_t y, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    GROUPED_SMALL("2");
}
__device__ __forceinline__ void mma_large_product(uint32_t d, uint32_t x, uint32_t y, uint32_t hi, uint32_t idesc) { GROUPED_LARGE("2"); }

// The lane that issues for a warp whose lanes all run the same code: with values that are the same in all lanes, instructions
// take them from uniform registers. An MMA issued so costs 37 cycles, from a branch that only one lane takes 104.
__device__ __forceinline__ bool elected() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// 16 contraction steps for one CTA with A in tensor memory, its parts AP columns apart, and B's parts below each other as one
// operand (idesc3: of three parts' columns, and so on): hi.[hi mid lo] to accumulators d0.., mid.[hi mid] to d1.., lo.[hi]
// to d2. accumulate == 0: the first overwrites all three. Called by the whole warp, `lead`: elected().
template <uint32_t AP>
__device__ __forceinline__ void mma_stacked_ts(uint32_t d0, uint32_t d1, uint32_t d2, uint32_t x, uint32_t y, uint32_t hi, uint32_t idesc3,
                                               uint32_t idesc2, uint32_t idesc1, uint32_t accumulate, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred p, t, q;\n\t.reg .b32 r, s;\n\t.reg .b64 db;\n\tsetp.ne.b32 q, %12, 0;\n\t"
        "setp.ne.b32 p, %9, 0;\n\tsetp.eq.b32 t, 0, 0;\n\tmov.b64 db, {%4, %5};\n\tadd.u32 r, %3, %10;\n\tadd.u32 s, %3, %11;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%3], db, %6, p;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%1], [r], db, %7, t;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%2], [s], db, %8, t;\n\t}"
        ::"r"(d0), "r"(d1), "r"(d2), "r"(x), "r"(y), "r"(hi), "r"(idesc3), "r"(idesc2), "r"(idesc1), "r"(accumulate), "n"(AP), "n"(2 * AP), "r"(lead)
        : "memory");
}

// The same sixteen steps as six products into one accumulator: B's parts bp units of 16 bytes apart, the five small products
// (accumulate == 0: the first overwrites the accumulator), and the large one.
#define GROUPED_TS(A, B, P) "mov.b64 db, {" B ", %4};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [" A "], db, %5, " P ";\n\t"
template <uint32_t AP>
__device__ __forceinline__ void mma_small_products_ts(uint32_t d, uint32_t x, uint32_t y, uint32_t bp, uint32_t hi, uint32_t idesc, uint32_t accumulate, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred p, t, q;\n\t.reg .b32 r, s, u, w;\n\t.reg .b64 db;\n\t"
        "setp.ne.b32 q, %9, 0;\n\tsetp.ne.b32 p, %6, 0;\n\tsetp.eq.b32 t, 0, 0;\n\tadd.u32 r, %1, %7;\n\tadd.u32 s, %1, %8;\n\tadd.u32 u, %2, %3;\n\tadd.u32 w, u, %3;\n\t"
        GROUPED_TS("s", "%2", "p") GROUPED_TS("%1", "w", "t") GROUPED_TS("r", "u", "t") GROUPED_TS("r", "%2", "t") GROUPED_TS("%1", "u", "t") "}"
        ::"r"(d), "r"(x), "r"(y), "r"(bp), "r"(hi), "r"(idesc), "r"(accumulate), "n"(AP), "n"(2 * AP), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void mma_large_product_ts(uint32_t d, uint32_t x, uint32_t y, uint32_t hi, uint32_t idesc, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred t, q;\n\t.reg .b64 db;\n\tsetp.ne.b32 q, %5, 0;\n\tsetp.eq.b32 t, 0, 0;\n\tmov.b64 db, {%2, %3};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, t;\n\t}"
        ::"r"(d), "r"(x), "r"(y), "r"(hi), "r"(idesc), "r"(lead)
        : "memory");
}

}  // namespace
}  // namespace tagi
