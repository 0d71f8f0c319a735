// Linear layers grouped by expert: rows [offsets[e], offsets[e + 1]) of the dispatch order go through expert e's weights.
// The offsets and the gather index are device data, so no pass waits for the host; both are checked where they are read
// (offsets are clamped to [0, S] and made non-decreasing, a row whose token lies outside [0, R) reads as zero).
#include "tagi_common.h"

namespace tagi {
namespace {

enum { FWD = 0, STATE = 1, PARAM = 2 };

struct GroupedArgs {
    int E, S, R, K, N;
    const int *offsets, *token;
    const float *mu_w, *var_w, *mu_b, *var_b, *a0, *a1, *jcb;  // a0, a1: activations (forward) or deltas; x: parameter pass
    const float *x;
    float *o0, *o1, *ob0, *ob1;
};

__device__ __forceinline__ void expert_rows(const GroupedArgs &a, int e, int &r0, int &r1) {
    r0 = min(max(__ldg(a.offsets + e), 0), a.S);
    r1 = min(max(__ldg(a.offsets + e + 1), r0), a.S);
}

// Input row of dispatch row p: -1 when its token is outside the tensor.
__device__ __forceinline__ int input_row(const GroupedArgs &a, int p) {
    const int r = a.token ? __ldg(a.token + p) : p;
    return (unsigned)r < (unsigned)a.R ? r : -1;
}

constexpr int TILE = 64, KT = 16;

// 64 x 64 tile of both outputs, 256 threads, 4 x 4 outputs each.
template <int PASS>
__global__ void __launch_bounds__(256) grouped_tile_kernel(const GroupedArgs a) {
    __shared__ float sa[2][KT][TILE + 1], sb[2][KT][TILE + 1];
    int e, r0, r1, m0;
    if (PASS == PARAM) {
        e = blockIdx.z;
        expert_rows(a, e, r0, r1);
        m0 = blockIdx.y * TILE;
    } else {
        int tile = blockIdx.x;
        for (e = 0; e < a.E; e++) {
            expert_rows(a, e, r0, r1);
            const int tiles = (r1 - r0 + TILE - 1) / TILE;
            if (tile < tiles) break;
            tile -= tiles;
        }
        if (e == a.E) return;
        m0 = r0 + tile * TILE;
    }
    const int c0 = (PASS == PARAM ? blockIdx.x : blockIdx.y) * TILE;
    const int depth = PASS == FWD ? a.K : PASS == STATE ? a.N : r1 - r0;
    const int rows = PASS == PARAM ? a.N : r1, cols = PASS == FWD ? a.N : a.K;
    const size_t wbase = (size_t)e * a.N * a.K;
    float acc0[4][4] = {}, acc1[4][4] = {};
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    for (int k0 = 0; k0 < depth; k0 += KT) {
        for (int i = threadIdx.x; i < TILE * KT; i += 256) {
            // consecutive threads run along the dimension that is contiguous in memory
            const int kk = PASS == PARAM ? i / TILE : i % KT, m = PASS == PARAM ? i % TILE : i / KT;
            float v0 = 0.f, v1 = 0.f;
            if (m0 + m < rows && k0 + kk < depth) {
                if (PASS == FWD) {
                    const int r = input_row(a, m0 + m);
                    if (r >= 0) v0 = __ldg(a.a0 + (size_t)r * a.K + k0 + kk), v1 = __ldg(a.a1 + (size_t)r * a.K + k0 + kk);
                } else if (PASS == STATE) {
                    v0 = __ldg(a.a0 + (size_t)(m0 + m) * a.N + k0 + kk);
                    v1 = __ldg(a.a1 + (size_t)(m0 + m) * a.N + k0 + kk);
                } else {
                    v0 = __ldg(a.a0 + (size_t)(r0 + k0 + kk) * a.N + m0 + m);
                    v1 = __ldg(a.a1 + (size_t)(r0 + k0 + kk) * a.N + m0 + m);
                }
            }
            sa[0][kk][m] = v0;
            sa[1][kk][m] = v1;
            const int kb = PASS == FWD ? i % KT : i / TILE, c = PASS == FWD ? i / KT : i % TILE;
            v0 = v1 = 0.f;
            if (c0 + c < cols && k0 + kb < depth) {
                if (PASS == FWD) {
                    v0 = __ldg(a.mu_w + wbase + (size_t)(c0 + c) * a.K + k0 + kb);
                    v1 = __ldg(a.var_w + wbase + (size_t)(c0 + c) * a.K + k0 + kb);
                } else if (PASS == STATE) {
                    v0 = __ldg(a.mu_w + wbase + (size_t)(k0 + kb) * a.K + c0 + c);
                } else {
                    const int r = input_row(a, r0 + k0 + kb);
                    if (r >= 0) v0 = __ldg(a.x + (size_t)r * a.K + c0 + c);
                }
            }
            sb[0][kb][c] = v0;
            sb[1][kb][c] = PASS == FWD ? v1 : v0 * v0;
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < KT; kk++) {
            float x[4], v[4], w[4], u[4];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                x[q] = sa[0][kk][ty * 4 + q], v[q] = sa[1][kk][ty * 4 + q];
                w[q] = sb[0][kk][tx * 4 + q], u[q] = sb[1][kk][tx * 4 + q];
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    acc0[i][j] += x[i] * w[j];
                    if (PASS == FWD) acc1[i][j] += v[i] * (w[j] * w[j]) + (x[i] * x[i] + v[i]) * u[j];
                    else acc1[i][j] += v[i] * u[j];
                }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int m = m0 + ty * 4 + i, c = c0 + tx * 4 + j;
            if (m >= rows || c >= cols) continue;
            float z = acc0[i][j], vz = acc1[i][j];
            if (PASS == FWD) {
                if (a.mu_b) z += __ldg(a.mu_b + (size_t)e * a.N + c), vz += __ldg(a.var_b + (size_t)e * a.N + c);
                a.o0[(size_t)m * a.N + c] = z;
                a.o1[(size_t)m * a.N + c] = vz;
            } else if (PASS == STATE) {
                const float q = a.jcb ? __ldg(a.jcb + (size_t)m * a.K + c) : 1.f;
                a.o0[(size_t)m * a.K + c] = z * q;
                a.o1[(size_t)m * a.K + c] = vz * q * q;
            } else {
                const size_t o = wbase + (size_t)m * a.K + c;
                const float s = __ldg(a.var_w + o);
                a.o0[o] = z * s;
                a.o1[o] = vz * s * s;
            }
        }
}

// dmu_b = var_b sum dmu_z, dvar_b = var_b^2 sum dvar_z over an expert's rows: 32 features x 8 groups of rows per CTA.
__global__ void __launch_bounds__(256) grouped_bias_kernel(const GroupedArgs a) {
    __shared__ float2 red[8][32];
    const int c = threadIdx.x & 31, g = threadIdx.x >> 5, n = blockIdx.x * 32 + c, e = blockIdx.y;
    int r0, r1;
    expert_rows(a, e, r0, r1);
    float s = 0.f, v = 0.f;
    if (n < a.N)
        for (int r = r0 + g; r < r1; r += 8) s += __ldg(a.a0 + (size_t)r * a.N + n), v += __ldg(a.a1 + (size_t)r * a.N + n);
    red[g][c] = make_float2(s, v);
    __syncthreads();
    if (g != 0 || n >= a.N) return;
    s = v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; k++) s += red[k][c].x, v += red[k][c].y;
    const float vb = __ldg(a.var_b + (size_t)e * a.N + n);
    a.ob0[(size_t)e * a.N + n] = vb * s;
    a.ob1[(size_t)e * a.N + n] = vb * vb * v;
}

inline int launched(const char *what) {
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? TAGI_OK : cuda_fail(e, what);
}

int check_grouped(const char *who, int E, int S, int K, int N, const int *offsets) {
    if (E < 1 || E > 1024 || S < 0 || K < 1 || N < 1)
        return fail(TAGI_ERR_INVALID_ARGUMENT, std::string(who) + ": 1 to 1024 experts, positive feature counts, rows must not be negative");
    if (K > (1 << 20) || N > (1 << 20) || S > (1 << 28))
        return fail(TAGI_ERR_INVALID_ARGUMENT, std::string(who) + ": more than 2^20 features or 2^28 rows");
    if (offsets == nullptr || !aligned4(offsets))
        return fail(TAGI_ERR_INVALID_ARGUMENT, std::string(who) + ": offsets is null or not 4-byte aligned");
    return TAGI_OK;
}

}  // namespace
}  // namespace tagi

using namespace tagi;

#define TAGI_PTR(p) TAGI_REQUIRE((p) != nullptr && aligned4(p), #p " is null or not 4-byte aligned")

extern "C" {

int tagi_grouped_linear_fwd(int E, int S, int R, int K, int N, int has_bias, const int *offsets, const int *token,
                            const float *mu_w, const float *var_w, const float *mu_b, const float *var_b, const float *mu_a,
                            const float *var_a, float *mu_z, float *var_z, void *stream) {
    int rc = check_grouped(__func__, E, S, K, N, offsets);
    if (rc != TAGI_OK) return rc;
    TAGI_PTR(mu_w);
    TAGI_PTR(var_w);
    if (has_bias) {
        TAGI_PTR(mu_b);
        TAGI_PTR(var_b);
    }
    TAGI_REQUIRE(token == nullptr || aligned4(token), "token is not 4-byte aligned");
    TAGI_REQUIRE(R >= 0, "input rows must not be negative");
    if (S == 0) return TAGI_OK;
    TAGI_REQUIRE(token != nullptr || R == S, "without a gather index the input has as many rows as the output");
    TAGI_REQUIRE(R > 0, "rows to compute but no input rows");
    TAGI_PTR(mu_a);
    TAGI_PTR(var_a);
    TAGI_PTR(mu_z);
    TAGI_PTR(var_z);
    GroupedArgs a{};
    a.E = E, a.S = S, a.R = R, a.K = K, a.N = N, a.offsets = offsets, a.token = token, a.mu_w = mu_w, a.var_w = var_w;
    a.mu_b = has_bias ? mu_b : nullptr, a.var_b = has_bias ? var_b : nullptr, a.a0 = mu_a, a.a1 = var_a, a.o0 = mu_z, a.o1 = var_z;
    grouped_tile_kernel<FWD><<<dim3(S / TILE + E, (N + TILE - 1) / TILE), 256, 0, static_cast<cudaStream_t>(stream)>>>(a);
    return launched("grouped_tile_kernel launch");
}

int tagi_grouped_linear_bwd_state(int E, int S, int K, int N, const int *offsets, const float *mu_w, const float *jcb,
                                  const float *dmu_z, const float *dvar_z, float *dmu_a, float *dvar_a, void *stream) {
    int rc = check_grouped(__func__, E, S, K, N, offsets);
    if (rc != TAGI_OK) return rc;
    TAGI_PTR(mu_w);
    TAGI_REQUIRE(jcb == nullptr || aligned4(jcb), "jcb is not 4-byte aligned");
    if (S == 0) return TAGI_OK;
    TAGI_PTR(dmu_z);
    TAGI_PTR(dvar_z);
    TAGI_PTR(dmu_a);
    TAGI_PTR(dvar_a);
    GroupedArgs a{};
    a.E = E, a.S = S, a.R = S, a.K = K, a.N = N, a.offsets = offsets, a.mu_w = mu_w, a.jcb = jcb, a.a0 = dmu_z, a.a1 = dvar_z;
    a.o0 = dmu_a, a.o1 = dvar_a;
    grouped_tile_kernel<STATE><<<dim3(S / TILE + E, (K + TILE - 1) / TILE), 256, 0, static_cast<cudaStream_t>(stream)>>>(a);
    return launched("grouped_tile_kernel launch");
}

int tagi_grouped_linear_bwd_param(int E, int S, int R, int K, int N, int has_bias, const int *offsets, const int *token,
                                  const float *var_w, const float *var_b, const float *mu_a, const float *dmu_z,
                                  const float *dvar_z, float *dmu_w, float *dvar_w, float *dmu_b, float *dvar_b, void *stream) {
    int rc = check_grouped(__func__, E, S, K, N, offsets);
    if (rc != TAGI_OK) return rc;
    TAGI_PTR(var_w);
    TAGI_PTR(dmu_w);
    TAGI_PTR(dvar_w);
    if (has_bias) {
        TAGI_PTR(var_b);
        TAGI_PTR(dmu_b);
        TAGI_PTR(dvar_b);
    }
    TAGI_REQUIRE(token == nullptr || aligned4(token), "token is not 4-byte aligned");
    TAGI_REQUIRE(R >= 0, "input rows must not be negative");
    if (S > 0) {
        TAGI_REQUIRE(token != nullptr || R == S, "without a gather index the input has as many rows as the deltas");
        TAGI_REQUIRE(R > 0, "deltas but no input rows");
        TAGI_PTR(mu_a);
        TAGI_PTR(dmu_z);
        TAGI_PTR(dvar_z);
    }
    GroupedArgs a{};
    a.E = E, a.S = S, a.R = R, a.K = K, a.N = N, a.offsets = offsets, a.token = token, a.var_w = var_w, a.x = mu_a;
    a.var_b = has_bias ? var_b : nullptr, a.a0 = dmu_z, a.a1 = dvar_z, a.o0 = dmu_w, a.o1 = dvar_w, a.ob0 = dmu_b, a.ob1 = dvar_b;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    grouped_tile_kernel<PARAM><<<dim3((K + TILE - 1) / TILE, (N + TILE - 1) / TILE, E), 256, 0, st>>>(a);
    rc = launched("grouped_tile_kernel launch");
    if (rc != TAGI_OK || !has_bias) return rc;
    grouped_bias_kernel<<<dim3((N + 31) / 32, E), 256, 0, st>>>(a);
    return launched("grouped_bias_kernel launch");
}

}  // extern "C"
