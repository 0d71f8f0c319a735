// Shared by the kernels of the Linear layers grouped by expert (tagi_grouped.cu, tagi_grouped_tc.cu).
#pragma once
#include "tagi_common.h"

namespace tagi {

enum { FWD = 0, STATE = 1, PARAM = 2 };

struct GroupedArgs {
    int E, S, R, K, N;
    int few;   // most rows of an expert for the kernels of tagi_grouped_few.cu
    const int *offsets, *token;
    // a0, a1: activations (forward) or deltas (backward); x: input means of the parameter pass
    const float *mu_w, *var_w, *mu_b, *var_b, *a0, *a1, *jcb, *x;
    // workspaces, 16-byte aligned: partial sums of the tiles that are cut; forward, mu_a^2 + var_a [R][K]
    float *parts, *second;
    float *o0, *o1, *ob0, *ob1;
};

#ifdef __CUDACC__
// Rows [r0, r1) of expert e. The offsets are device data: whatever they hold, the rows lie in [0, S].
__device__ __forceinline__ void expert_rows(const GroupedArgs &a, int e, int &r0, int &r1) {
    r0 = min(max(__ldg(a.offsets + e), 0), a.S);
    r1 = min(max(__ldg(a.offsets + e + 1), r0), a.S);
}

// Input row of dispatch row p: -1 when its token is outside the tensor.
__device__ __forceinline__ int input_row(const GroupedArgs &a, int p) {
    const int r = a.token ? __ldg(a.token + p) : p;
    return (unsigned)r < (unsigned)a.R ? r : -1;
}

__device__ __forceinline__ uint32_t smem_at(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
// floats of p's 16-byte group of memory before p
__device__ __forceinline__ int shift_of(const float *p) { return (int)((unsigned long long)p >> 2) & 3; }
// The 16-byte group of memory at src, of whose floats `left` lie before the row's end; zeros behind it.
__device__ __forceinline__ void copy_group(float *dst, const float *src, int left) {
    if (left > 0)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_at(dst)), "l"(src), "r"(left < 4 ? left * 4 : 16) : "memory");
    else
        *reinterpret_cast<float4 *>(dst) = make_float4(0.f, 0.f, 0.f, 0.f);
}
__device__ __forceinline__ void copy_float(float *dst, const float *src, bool in) {
    if (in) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_at(dst)), "l"(src) : "memory");
    else *dst = 0.f;
}
// A group that begins before its tensor does, `before` floats: only the floats of the tensor.
__device__ __forceinline__ void copy_first_group(float *dst, const float *src, int before, int left) {
    for (int c = before; c < 4; c++) copy_float(dst + c, src + c, c < left);
}
#endif

// Which kernel an expert's rows run on, decided on the device by their number (few: see GroupedArgs):
//   up to few           tagi_grouped_few.cu   one pass over the weights on the FP32 pipe
//   up to THIN_ROWS     tagi_grouped_thin.cu  tensor cores, tiles of 128 features (forward and state pass)
//   up to MIDDLE_ROWS   the same for up to 128 rows, if middle_likely()
//   more                tagi_grouped_tc.cu    tensor cores, tiles of 256 features x up to 256 rows
// Measured on eight experts of 4096 x 4096, forward pass, 4 / 8 / 16 / 32 rows each: few 220 / 317 / 522 / 936 us; thin 279 / 314 /
// 337 us at 16 / 32 / 40; 56 / 100 / 128 rows: middle 494 / 524 / 583 us, the wide kernel 813 / 843 / 862 us. (Of 1001 x 1001, 7 rows:
// few 48, thin 70 us.) Parameter pass at 7 / 10 / 14 / 20 rows: few
// 377 / 419 / 486 / 595 us, the wide kernel 503 to 507 us.
constexpr int FEW_ROWS = 8, FEW_PARAM_ROWS = 14, THIN_ROWS = 48, MIDDLE_ROWS = 128;

// The middle kernel is tried where the average expert makes 49 to 128 rows likely: one that finds nothing to do takes up to 7 us.
inline bool middle_likely(int E, int S) { return S > THIN_ROWS && S > THIN_ROWS / 2 * E && S <= (MIDDLE_ROWS + 32) * E; }

// the rows that a pass reads (of weights, activations and deltas) are whole 16-byte groups
inline bool grouped_aligned(int pass, const GroupedArgs &a) {
    return a.K % 4 == 0 && (pass == FWD || a.N % 4 == 0) && (pass == PARAM || (aligned16(a.mu_w) && aligned16(a.var_w))) && aligned16(a.a0) &&
           aligned16(a.a1) && aligned16(a.x);
}

// mu_a^2 + var_a of every input row to a.second, for the tensor-core kernels
int grouped_second_moment(const GroupedArgs &a, cudaStream_t st);
int grouped_few(int pass, const GroupedArgs &a, cudaStream_t st);
int grouped_thin(int pass, const GroupedArgs &a, cudaStream_t st);
size_t grouped_thin_parts_bytes(int pass, int E, int S, int K, int N);   // forward and state pass
int grouped_thin_status(int *out, int reset);
int grouped_tc(int pass, const GroupedArgs &a, cudaStream_t st);
int grouped_tc_pairs(int pass, int E, int S, int K, int N);
size_t grouped_tc_parts_bytes(int pass, int E, int S, int K, int N);

}  // namespace tagi
