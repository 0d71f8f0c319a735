// Shared by the kernels of the Linear layers grouped by expert (tagi_grouped.cu, tagi_grouped_tc.cu).
#pragma once
#include "tagi_common.h"

namespace tagi {

enum { FWD = 0, STATE = 1, PARAM = 2 };

struct GroupedArgs {
    int E, S, R, K, N;
    const int *offsets, *token;
    // a0, a1: activations (forward) or deltas (backward); x: input means of the parameter pass
    const float *mu_w, *var_w, *mu_b, *var_b, *a0, *a1, *jcb, *x;
    float *second;   // forward: workspace for mu_a^2 + var_a, [R][K], 16-byte aligned
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
#endif

// Experts with up to this many rows run on the kernels of tagi_grouped_few.cu (one pass over the weights on the FP32 pipe),
// those with more on the tensor cores.
constexpr int FEW_ROWS = 32;

int grouped_few(int pass, const GroupedArgs &a, cudaStream_t st);
int grouped_tc(int pass, const GroupedArgs &a, cudaStream_t st);

}  // namespace tagi
