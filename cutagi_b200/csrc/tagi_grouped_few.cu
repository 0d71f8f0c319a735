// Linear layers grouped by expert, experts with few rows: every weight is read once and met by all rows of its expert, on
// the FP32 pipe. These passes are bound by HBM (8, 4 and 12 bytes a weight in the forward, state and parameter pass), as
// long as the rows' multiplications keep up: 3, 2 and 2 a weight and row. Experts with more rows than the limits below are
// left to the tensor-core kernel, which in turn leaves these alone; the offsets are device data, so both are launched when
// the number of rows in all does not rule one out.
#include "tagi_grouped.h"

namespace tagi {
namespace {

constexpr unsigned FULL = 0xffffffffu;

// W consecutive floats. Weights pass by once: they are kept out of L1, where the rows are wanted.
template <int W>
__device__ __forceinline__ void load(const float *p, float (&v)[W]) {
    if (W == 4) {
        const float4 t = __ldg(reinterpret_cast<const float4 *>(p));
        v[0] = t.x, v[1 % W] = t.y, v[2 % W] = t.z, v[3 % W] = t.w;
    } else {
        v[0] = __ldg(p);
    }
}
template <int W>
__device__ __forceinline__ void load_once(const float *p, float (&v)[W]) {
    if (W == 4)
        asm("ld.global.nc.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];"
            : "=f"(v[0]), "=f"(v[1 % W]), "=f"(v[2 % W]), "=f"(v[3 % W])
            : "l"(p));
    else
        asm("ld.global.nc.L1::no_allocate.f32 %0, [%1];" : "=f"(v[0]) : "l"(p));
}
template <int W>
__device__ __forceinline__ void zero(float (&v)[W]) {
#pragma unroll
    for (int c = 0; c < W; c++) v[c] = 0.f;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}

// ---------------------------------------------------------------------------------------------------------- forward
// A warp computes FEATURES output features of R rows, its lanes along the contraction.
constexpr int FEATURES = 4, FWD_WARPS = 8;

template <int W, int R>
__device__ __forceinline__ void forward_rows(const GroupedArgs &a, int e, int r0, int rows, int n0) {
    const int lane = threadIdx.x & 31;
    float z[FEATURES][R], vz[FEATURES][R];
#pragma unroll
    for (int f = 0; f < FEATURES; f++)
#pragma unroll
        for (int r = 0; r < R; r++) z[f][r] = vz[f][r] = 0.f;
    int row[R];
#pragma unroll
    for (int r = 0; r < R; r++) row[r] = r < rows ? input_row(a, r0 + r) : -1;
    const size_t w0 = ((size_t)e * a.N + n0) * a.K;
#pragma unroll 1
    for (int k = lane * W; k < a.K; k += 32 * W) {
        float w[FEATURES][W], vw[FEATURES][W];
#pragma unroll
        for (int f = 0; f < FEATURES; f++) {
            zero(w[f]), zero(vw[f]);
            if (n0 + f < a.N) {
                load_once<W>(a.mu_w + w0 + (size_t)f * a.K + k, w[f]);
                load_once<W>(a.var_w + w0 + (size_t)f * a.K + k, vw[f]);
            }
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
            float x[W], v[W];
            zero(x), zero(v);
            if (row[r] >= 0) {
                load<W>(a.a0 + (size_t)row[r] * a.K + k, x);
                load<W>(a.a1 + (size_t)row[r] * a.K + k, v);
            }
#pragma unroll
            for (int c = 0; c < W; c++) {
                const float s = fmaf(x[c], x[c], v[c]);
#pragma unroll
                for (int f = 0; f < FEATURES; f++) {
                    z[f][r] = fmaf(x[c], w[f][c], z[f][r]);
                    vz[f][r] = fmaf(s, vw[f][c], fmaf(v[c], w[f][c] * w[f][c], vz[f][r]));
                }
            }
        }
    }
#pragma unroll
    for (int f = 0; f < FEATURES; f++)
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float m = warp_sum(z[f][r]), v = warp_sum(vz[f][r]);
            const int n = n0 + f;
            if (lane == (f * R + r) % 32 && n < a.N && r < rows) {
                const size_t o = (size_t)(r0 + r) * a.N + n;
                a.o0[o] = m + (a.mu_b ? __ldg(a.mu_b + (size_t)e * a.N + n) : 0.f);
                a.o1[o] = v + (a.mu_b ? __ldg(a.var_b + (size_t)e * a.N + n) : 0.f);
            }
        }
}

template <int W>
__global__ void __launch_bounds__(FWD_WARPS * 32) grouped_few_fwd_kernel(const GroupedArgs a) {
    const int e = blockIdx.y, n0 = (blockIdx.x * FWD_WARPS + (threadIdx.x >> 5)) * FEATURES;
    int r0, r1;
    expert_rows(a, e, r0, r1);
    const int rows = r1 - r0;
    if (rows == 0 || rows > FEW_ROWS || n0 >= a.N) return;
    if (rows == 1) forward_rows<W, 1>(a, e, r0, rows, n0);
    else if (rows == 2) forward_rows<W, 2>(a, e, r0, rows, n0);
    else if (rows <= 4) forward_rows<W, 4>(a, e, r0, rows, n0);
    else forward_rows<W, 8>(a, e, r0, rows, n0);
}

// ------------------------------------------------------------------------------------------------------------ state
// A CTA computes 64 input features of R rows: 16 lanes of four features each, the contraction over the output features cut
// among the 32 half-warps of 16 warps, whose sums are then added in a fixed order.
constexpr int STATE_WARPS = 16, STATE_COLS = 64;

template <int W, int R>
__device__ __forceinline__ void state_rows(const GroupedArgs &a, int e, int r0, int rows, float *red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp * 2 + (lane >> 4);
    const int k = blockIdx.x * STATE_COLS + (lane & 15) * 4;
    float d[R][4], v[R][4];
#pragma unroll
    for (int r = 0; r < R; r++) zero(d[r]), zero(v[r]);
    // W == 4: four output features at a time, k .. k + 3 all inside or all outside
    for (int n = part * W; n < a.N; n += 2 * STATE_WARPS * W) {
        float w[W][4];
#pragma unroll
        for (int i = 0; i < W; i++) {
            zero(w[i]);
            const float *p = a.mu_w + ((size_t)e * a.N + n + i) * a.K + k;
            if (W == 4) {
                if (k < a.K) load_once<4>(p, w[i]);
            } else {
#pragma unroll
                for (int c = 0; c < 4; c++)
                    if (k + c < a.K) w[i][c] = __ldg(p + c);
            }
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
            float x[W], y[W];
            zero(x), zero(y);
            if (r < rows) {
                load<W>(a.a0 + (size_t)(r0 + r) * a.N + n, x);
                load<W>(a.a1 + (size_t)(r0 + r) * a.N + n, y);
            }
#pragma unroll
            for (int i = 0; i < W; i++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    d[r][c] = fmaf(x[i], w[i][c], d[r][c]);
                    v[r][c] = fmaf(y[i], w[i][c] * w[i][c], v[r][c]);
                }
        }
    }
    // the halves of a warp, then the warps, one row at a time: red holds [STATE_WARPS][2][64]
#pragma unroll
    for (int r = 0; r < R; r++) {
        if (r >= rows) break;
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const float s = d[r][c] + __shfl_xor_sync(FULL, d[r][c], 16), t = v[r][c] + __shfl_xor_sync(FULL, v[r][c], 16);
            if (lane < 16) {
                red[warp * 128 + lane * 4 + c] = s;
                red[warp * 128 + 64 + lane * 4 + c] = t;
            }
        }
        __syncthreads();
        if (threadIdx.x < 128) {
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < STATE_WARPS; w++) s += red[w * 128 + threadIdx.x];
            const int col = blockIdx.x * STATE_COLS + (threadIdx.x & 63);
            if (col < a.K) {
                const size_t o = (size_t)(r0 + r) * a.K + col;
                const float j = a.jcb ? __ldg(a.jcb + o) : 1.f;
                if (threadIdx.x < 64) a.o0[o] = s * j;
                else a.o1[o] = s * j * j;
            }
        }
    }
}

template <int W>
__global__ void __launch_bounds__(STATE_WARPS * 32) grouped_few_state_kernel(const GroupedArgs a) {
    __shared__ float red[STATE_WARPS * 128];
    const int e = blockIdx.y;
    int r0, r1;
    expert_rows(a, e, r0, r1);
    const int rows = r1 - r0;
    if (rows == 0 || rows > FEW_ROWS) return;
    if (rows == 1) state_rows<W, 1>(a, e, r0, rows, red);
    else if (rows == 2) state_rows<W, 2>(a, e, r0, rows, red);
    else if (rows <= 4) state_rows<W, 4>(a, e, r0, rows, red);
    else state_rows<W, 8>(a, e, r0, rows, red);
}

// -------------------------------------------------------------------------------------------------------- parameters
// A warp computes PARAM_N output features x 32 lanes of W input features; a CTA stacks 8 warps along the output features.
constexpr int PARAM_N = 8, PARAM_WARPS = 8;

template <int W>
__global__ void __launch_bounds__(PARAM_WARPS * 32) grouped_few_param_kernel(const GroupedArgs a) {
    const int e = blockIdx.z;
    int r0, r1;
    expert_rows(a, e, r0, r1);
    if (r1 - r0 > FEW_PARAM_ROWS) return;
    const int lane = threadIdx.x & 31, block_n = blockIdx.y * PARAM_WARPS * PARAM_N, n0 = block_n + (threadIdx.x >> 5) * PARAM_N;
    const int k = (blockIdx.x * 32 + lane) * W;
    if (a.var_b && blockIdx.x == 0 && threadIdx.x < PARAM_WARPS * PARAM_N && block_n + threadIdx.x < a.N) {
        const int n = block_n + threadIdx.x;
        float s = 0.f, t = 0.f;
        for (int r = r0; r < r1; r++) s += __ldg(a.a0 + (size_t)r * a.N + n), t += __ldg(a.a1 + (size_t)r * a.N + n);
        const float vb = __ldg(a.var_b + (size_t)e * a.N + n);
        a.ob0[(size_t)e * a.N + n] = vb * s;
        a.ob1[(size_t)e * a.N + n] = vb * vb * t;
    }
    if (n0 >= a.N || k >= a.K) return;
    float d[PARAM_N][W], v[PARAM_N][W], s[PARAM_N][W];
    const size_t o = ((size_t)e * a.N + n0) * a.K + k;
#pragma unroll
    for (int i = 0; i < PARAM_N; i++) {
        zero(d[i]), zero(v[i]), zero(s[i]);
        if (n0 + i < a.N) load_once<W>(a.var_w + o + (size_t)i * a.K, s[i]);   // on their way while the rows are added up
    }
    for (int r = r0; r < r1; r++) {
        const int row = input_row(a, r);
        if (row < 0) continue;
        float x[W], q[W];
        load<W>(a.x + (size_t)row * a.K + k, x);
#pragma unroll
        for (int c = 0; c < W; c++) q[c] = x[c] * x[c];
#pragma unroll
        for (int i = 0; i < PARAM_N; i++) {
            if (n0 + i >= a.N) break;
            const float dm = __ldg(a.a0 + (size_t)r * a.N + n0 + i), dv = __ldg(a.a1 + (size_t)r * a.N + n0 + i);
#pragma unroll
            for (int c = 0; c < W; c++) d[i][c] = fmaf(dm, x[c], d[i][c]), v[i][c] = fmaf(dv, q[c], v[i][c]);
        }
    }
#pragma unroll
    for (int i = 0; i < PARAM_N; i++) {
        if (n0 + i >= a.N) break;
#pragma unroll
        for (int c = 0; c < W; c++) d[i][c] *= s[i][c], v[i][c] *= s[i][c] * s[i][c];
        float *p = a.o0 + o + (size_t)i * a.K, *u = a.o1 + o + (size_t)i * a.K;
        if (W == 4) {
            *reinterpret_cast<float4 *>(p) = make_float4(d[i][0], d[i][1 % W], d[i][2 % W], d[i][3 % W]);
            *reinterpret_cast<float4 *>(u) = make_float4(v[i][0], v[i][1 % W], v[i][2 % W], v[i][3 % W]);
        } else {
            *p = d[i][0];
            *u = v[i][0];
        }
    }
}

}  // namespace

int grouped_few(int pass, const GroupedArgs &a, cudaStream_t st) {
    const bool k4 = a.K % 4 == 0, n4 = a.N % 4 == 0;
    if (pass == FWD) {
        const dim3 grid((a.N + FWD_WARPS * FEATURES - 1) / (FWD_WARPS * FEATURES), a.E);
        if (k4 && aligned16(a.mu_w) && aligned16(a.var_w) && aligned16(a.a0) && aligned16(a.a1))
            grouped_few_fwd_kernel<4><<<grid, FWD_WARPS * 32, 0, st>>>(a);
        else
            grouped_few_fwd_kernel<1><<<grid, FWD_WARPS * 32, 0, st>>>(a);
    } else if (pass == STATE) {
        const dim3 grid((a.K + STATE_COLS - 1) / STATE_COLS, a.E);
        if (k4 && n4 && aligned16(a.mu_w) && aligned16(a.a0) && aligned16(a.a1))
            grouped_few_state_kernel<4><<<grid, STATE_WARPS * 32, 0, st>>>(a);
        else
            grouped_few_state_kernel<1><<<grid, STATE_WARPS * 32, 0, st>>>(a);
    } else {
        const bool vec = k4 && aligned16(a.var_w) && aligned16(a.x) && aligned16(a.o0) && aligned16(a.o1);
        const dim3 grid((a.K + 32 * (vec ? 4 : 1) - 1) / (32 * (vec ? 4 : 1)), (a.N + PARAM_WARPS * PARAM_N - 1) / (PARAM_WARPS * PARAM_N), a.E);
        if (vec) grouped_few_param_kernel<4><<<grid, PARAM_WARPS * 32, 0, st>>>(a);
        else grouped_few_param_kernel<1><<<grid, PARAM_WARPS * 32, 0, st>>>(a);
    }
    TAGI_CUDA(cudaGetLastError());
    return TAGI_OK;
}

}  // namespace tagi
