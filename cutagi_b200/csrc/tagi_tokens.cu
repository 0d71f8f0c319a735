// Layers of token models on (mean, variance) rows: LayerNorm over a row's features, the combination of a token's expert
// rows and its backward pass, and the sum of the state deltas over the experts that a token was sent to. All of them are
// HBM-bound: every tensor is read or written once.
#include "tagi_common.h"

#include <type_traits>

namespace tagi {
namespace {

constexpr int MAX_ROWS = 1 << 30, MAX_FEATURES = 1 << 24;   // what the kernels' and launches' 32-bit counts hold

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sums of two values over the TPR threads that share a row, result in every one of them. TPR is a multiple of 32; `red`
// holds two floats per warp of the CTA. The leading barrier lets `red` be used again.
template <int TPR>
__device__ __forceinline__ void row_sum2(float &a, float &b, float2 *red) {
    a = warp_sum(a);
    b = warp_sum(b);
    if (TPR == 32) return;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    const int w0 = (threadIdx.x / TPR) * (TPR / 32);
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < TPR / 32; w++) a += red[w0 + w].x, b += red[w0 + w].y;
}

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
__device__ __forceinline__ void store(float *p, const float (&v)[W]) {
    if (W == 4) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1 % W], v[2 % W], v[3 % W]);
    else *p = v[0];
}

// ------------------------------------------------------------------------------------------------------- LayerNorm

constexpr int LN_EPT = 16;     // elements of a row that a thread keeps in registers
constexpr int LN_KEPT = LN_EPT * 1024;  // longest row that one CTA keeps

struct LnArgs {
    int R, n;
    float eps;
    const float *mu_w, *var_w, *mu_b, *var_b, *mu_a, *var_a;
    float *mu_row, *var_row, *mu_z, *var_z;
};

template <int W>
__device__ __forceinline__ void ln_apply(const LnArgs &a, int i, float mean, float inv, const float (&x)[W],
                                         const float (&v)[W], float *mz, float *vz) {
    float w[W], vw[W], mb[W], vb[W], z[W], s[W];
    load<W>(a.mu_w + i, w);
    load<W>(a.var_w + i, vw);
    if (a.mu_b) {
        load<W>(a.mu_b + i, mb);
        load<W>(a.var_b + i, vb);
    }
#pragma unroll
    for (int c = 0; c < W; c++) {
        const float t = x[c] - mean;
        z[c] = inv * t * w[c] + (a.mu_b ? mb[c] : 0.f);
        s[c] = inv * inv * (v[c] * (w[c] * w[c] + vw[c]) + vw[c] * t * t) + (a.mu_b ? vb[c] : 0.f);
    }
    store<W>(mz, z);
    store<W>(vz, s);
}

// TPR threads share a row of at most 16 * TPR features, which stays in their registers between the statistics and the
// normalisation: mu_a and var_a are read once. W = 4: rows are multiples of four floats and 16-byte aligned.
template <int W, int TPR>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) ln_fwd_kernel(const LnArgs a) {
    __shared__ float2 red[32];
    constexpr int THREADS = TPR < 256 ? 256 : TPR, ROWS = THREADS / TPR, G = LN_EPT / W;
    const long r = (long)blockIdx.x * ROWS + threadIdx.x / TPR;
    const int t = threadIdx.x % TPR;
    const bool live = r < a.R;
    const float *mu = a.mu_a + r * a.n, *var = a.var_a + r * a.n;
    float x[G][W], v[G][W], s = 0.f, sv = 0.f;
#pragma unroll
    for (int g = 0; g < G; g++) {
        const int i = (g * TPR + t) * W;
#pragma unroll
        for (int c = 0; c < W; c++) x[g][c] = v[g][c] = 0.f;
        if (live && i < a.n) {
            load<W>(mu + i, x[g]);
            load<W>(var + i, v[g]);
        }
#pragma unroll
        for (int c = 0; c < W; c++) s += x[g][c], sv += v[g][c];
    }
    row_sum2<TPR>(s, sv, red);
    const float mean = s / a.n;
    float m2 = 0.f, none = 0.f;
#pragma unroll
    for (int g = 0; g < G; g++)
        if ((g * TPR + t) * W < a.n) {
#pragma unroll
            for (int c = 0; c < W; c++) m2 += (x[g][c] - mean) * (x[g][c] - mean);
        }
    row_sum2<TPR>(m2, none, red);
    const float var_row = (m2 + sv) / (a.n - 1), inv = 1.0f / sqrtf(var_row + a.eps);
    if (!live) return;
    if (t == 0) a.mu_row[r] = mean, a.var_row[r] = var_row;
#pragma unroll
    for (int g = 0; g < G; g++) {
        const int i = (g * TPR + t) * W;
        if (i < a.n) ln_apply<W>(a, i, mean, inv, x[g], v[g], a.mu_z + r * a.n + i, a.var_z + r * a.n + i);
    }
}

// Rows longer than a CTA can keep: three passes over the row, the second and third from L2.
template <int W>
__global__ void __launch_bounds__(1024) ln_fwd_long_kernel(const LnArgs a) {
    __shared__ float2 red[32];
    const long r = blockIdx.x;
    const float *mu = a.mu_a + r * a.n, *var = a.var_a + r * a.n;
    float s = 0.f, sv = 0.f, m2 = 0.f, none = 0.f, x[W], v[W];
    for (long i = (long)threadIdx.x * W; i < a.n; i += 1024 * W) {
        load<W>(mu + i, x);
        load<W>(var + i, v);
#pragma unroll
        for (int c = 0; c < W; c++) s += x[c], sv += v[c];
    }
    row_sum2<1024>(s, sv, red);
    const float mean = s / a.n;
    for (long i = (long)threadIdx.x * W; i < a.n; i += 1024 * W) {
        load<W>(mu + i, x);
#pragma unroll
        for (int c = 0; c < W; c++) m2 += (x[c] - mean) * (x[c] - mean);
    }
    row_sum2<1024>(m2, none, red);
    const float var_row = (m2 + sv) / (a.n - 1), inv = 1.0f / sqrtf(var_row + a.eps);
    if (threadIdx.x == 0) a.mu_row[r] = mean, a.var_row[r] = var_row;
    for (long i = (long)threadIdx.x * W; i < a.n; i += 1024 * W) {
        load<W>(mu + i, x);
        load<W>(var + i, v);
        ln_apply<W>(a, (int)i, mean, inv, x, v, a.mu_z + r * a.n + i, a.var_z + r * a.n + i);
    }
}

struct LnBwdArgs {
    int R, n, chunk;
    float eps;
    const float *mu_w, *var_w, *var_b, *mu_a, *jcb, *mu_row, *var_row, *dmu_o, *dvar_o;
    float *dmu, *dvar, *dmu_w, *dvar_w, *dmu_b, *dvar_b;
    float *part;  // [chunks][4][n], or null: one chunk, results written directly
};

constexpr int LN_BWD_THREADS = 128;

// State deltas and the sums over a chunk of rows for four columns a thread: neighbours (W = 4), or U that are 128 apart (W = 1:
// rows of an odd length start anywhere, but as many loads are on their way). The parameter deltas' factors of var_w and var_b
// do not depend on the row: they are applied to the sums. 16384 rows of 1001: 66 us with U = 4, 76 us with U = 1; of 75: 17 and
// 15 us.
template <int W, int U>
__global__ void __launch_bounds__(LN_BWD_THREADS) ln_bwd_kernel(const LnBwdArgs a) {
    const int i0 = blockIdx.x * LN_BWD_THREADS * W * U + threadIdx.x * W;
    if (i0 >= a.n) return;
    const long r0 = (long)blockIdx.y * a.chunk, r1 = min((long)a.R, r0 + a.chunk);
    float w[U][W], s0[U][W], s1[U][W], s2[U][W], s3[U][W];
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (U == 1 || i0 + u * LN_BWD_THREADS < a.n) load<W>(a.mu_w + i0 + u * LN_BWD_THREADS, w[u]);
#pragma unroll
        for (int c = 0; c < W; c++) s0[u][c] = s1[u][c] = s2[u][c] = s3[u][c] = 0.f;
    }
#pragma unroll(U == 1 ? 2 : 1)
    for (long r = r0; r < r1; r++) {
        const float inv = 1.0f / sqrtf(__ldg(a.var_row + r) + a.eps), mean = __ldg(a.mu_row + r);
        float x[U][W], dm[U][W], dv[U][W], j[U][W];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long at = r * a.n + i0 + u * LN_BWD_THREADS;
            if (U == 1 || i0 + u * LN_BWD_THREADS < a.n) {
                load<W>(a.mu_a + at, x[u]);
                load<W>(a.dmu_o + at, dm[u]);
                load<W>(a.dvar_o + at, dv[u]);
                if (a.jcb) load<W>(a.jcb + at, j[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (U > 1 && i0 + u * LN_BWD_THREADS >= a.n) continue;
            float o[W], p[W];
#pragma unroll
            for (int c = 0; c < W; c++) {
                const float z = inv * (x[u][c] - mean), t = inv * w[u][c] * (a.jcb ? j[u][c] : 1.f);
                s0[u][c] += z * dm[u][c];
                s1[u][c] += z * dv[u][c] * z;
                s2[u][c] += dm[u][c];
                s3[u][c] += dv[u][c];
                o[c] = t * dm[u][c];
                p[c] = t * dv[u][c] * t;
            }
            if (a.dmu) {
                store<W>(a.dmu + r * a.n + i0 + u * LN_BWD_THREADS, o);
                store<W>(a.dvar + r * a.n + i0 + u * LN_BWD_THREADS, p);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i = i0 + u * LN_BWD_THREADS;
        if (U > 1 && i >= a.n) continue;
        if (a.part) {
            float *q = a.part + (size_t)blockIdx.y * 4 * a.n + i;
#pragma unroll
            for (int c = 0; c < W; c++) q[c] = s0[u][c], q[a.n + c] = s1[u][c], q[2L * a.n + c] = s2[u][c], q[3L * a.n + c] = s3[u][c];
        } else {
#pragma unroll
            for (int c = 0; c < W; c++) {
                const float vw = __ldg(a.var_w + i + c);
                a.dmu_w[i + c] = vw * s0[u][c];
                a.dvar_w[i + c] = vw * vw * s1[u][c];
                if (a.var_b) {
                    const float vb = __ldg(a.var_b + i + c);
                    a.dmu_b[i + c] = vb * s2[u][c];
                    a.dvar_b[i + c] = vb * vb * s3[u][c];
                }
            }
        }
    }
}

// Sum of the chunks' partials in a fixed order: 32 columns x 32 groups of chunks per CTA, one of the four sums per blockIdx.y
constexpr int FINAL_GROUPS = 32;
__global__ void __launch_bounds__(FINAL_GROUPS * 32) ln_bwd_final_kernel(const LnBwdArgs a, int chunks) {
    __shared__ float red[FINAL_GROUPS][33];
    const int c = threadIdx.x & 31, g = threadIdx.x >> 5, i = blockIdx.x * 32 + c, q = blockIdx.y;
    float s = 0.f;
    if (i < a.n)
#pragma unroll 4
        for (int k = g; k < chunks; k += FINAL_GROUPS) s += __ldg(a.part + ((size_t)k * 4 + q) * a.n + i);
    red[g][c] = s;
    __syncthreads();
    if (g != 0 || i >= a.n) return;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < FINAL_GROUPS; k++) s += red[k][c];
    const float *f = q < 2 ? a.var_w : a.var_b;
    const float v = __ldg(f + i);
    float *o = q == 0 ? a.dmu_w : q == 1 ? a.dvar_w : q == 2 ? a.dmu_b : a.dvar_b;
    o[i] = (q & 1) ? v * v * s : v * s;
}

inline int launched(const char *what) {
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? TAGI_OK : cuda_fail(e, what);
}

template <int W>
int ln_fwd_launch(const LnArgs &a, cudaStream_t st) {
    if (a.n > LN_KEPT) ln_fwd_long_kernel<W><<<a.R, 1024, 0, st>>>(a);
    else if (a.n > 16 * 512) ln_fwd_kernel<W, 1024><<<a.R, 1024, 0, st>>>(a);
    else if (a.n > 16 * 256) ln_fwd_kernel<W, 512><<<a.R, 512, 0, st>>>(a);
    else if (a.n > 16 * 128) ln_fwd_kernel<W, 256><<<a.R, 256, 0, st>>>(a);
    else if (a.n > 16 * 64) ln_fwd_kernel<W, 128><<<(a.R + 1) / 2, 256, 0, st>>>(a);
    else if (a.n > 16 * 32) ln_fwd_kernel<W, 64><<<(a.R + 3) / 4, 256, 0, st>>>(a);
    else ln_fwd_kernel<W, 32><<<(a.R + 7) / 8, 256, 0, st>>>(a);
    return launched("ln_fwd_kernel launch");
}

bool all16(std::initializer_list<const void *> ps) {
    for (const void *p : ps)
        if (p && !aligned16(p)) return false;
    return true;
}

// How the rows are cut into chunks whose partial sums are added afterwards: enough CTAs to keep eight per SM busy, at
// least 16 rows in each (a chunk costs 16 bytes a column of partials against 20 to 24 a row).
int ln_bwd_chunk(int R, int n) {
    const long tiles = (n + LN_BWD_THREADS * 4 - 1) / (LN_BWD_THREADS * 4), want = (148 * 8 + tiles - 1) / tiles;
    const long chunk = (R + want - 1) / want;
    return (int)(chunk < 16 ? 16 : chunk);
}
int ln_bwd_chunks(int R, int n) { return R == 0 ? 0 : (R + ln_bwd_chunk(R, n) - 1) / ln_bwd_chunk(R, n); }

// ------------------------------------------------------------------------------------------- combination of expert rows

struct CombineArgs {
    int T, k, N, S;
    const int *pos;
    const float *mu_g, *var_g, *mu_x, *var_x, *jcb;
    float *mu_y, *var_y;
};

// Row of slot j of token t, or -1: entries that name no row of [0, S) have none.
__device__ __forceinline__ int slot_row(const int *pos, long i, int S) {
    const int p = __ldg(pos + i);
    return (unsigned)p < (unsigned)S ? p : -1;
}

constexpr int SLOTS = 4;   // of a token that are worked on together

// GATED: mu = sum g x, var = sum var_g (x^2 + var_x) + g^2 var_x. Otherwise mu = J sum x, var = J^2 sum var_x.
// TPR threads share a token, four features each at a time: consecutive ones (W = 4), or TPR apart (W = 1: rows of an odd
// length start anywhere, but four loads are on their way all the same).
template <int W, int TPR, bool GATED>
__global__ void __launch_bounds__(256, W == 4 || !GATED ? 8 : 6) combine_fwd_kernel(const CombineArgs a) {
    constexpr int U = 4 / W;
    const unsigned tiles = (a.N + 4 * TPR - 1) / (4 * TPR);   // one, unless TPR is 256
    const long t = (long)(blockIdx.x / tiles) * (256 / TPR) + threadIdx.x / TPR;
    const int i0 = (int)(blockIdx.x % tiles) * 4 * TPR + threadIdx.x % TPR * W;
    if (t >= a.T || i0 >= a.N) return;
    float m[U][W], s[U][W];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int c = 0; c < W; c++) m[u][c] = s[u][c] = 0.f;
    // few registers and many threads: fetching the rows of four slots before the first is used was slower (141 against 123 us)
#pragma unroll(W == 4 ? 4 : 2)
    for (int j = 0; j < a.k; j++) {
        const int p = slot_row(a.pos, t * a.k + j, a.S);
        if (p < 0) continue;
        float x[U][W], v[U][W];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i0 + u * TPR < a.N) {
                load<W>(a.mu_x + (long)p * a.N + i0 + u * TPR, x[u]);
                load<W>(a.var_x + (long)p * a.N + i0 + u * TPR, v[u]);
            }
        const float g = GATED ? __ldg(a.mu_g + t * a.k + j) : 1.f, vg = GATED ? __ldg(a.var_g + t * a.k + j) : 0.f;
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i0 + u * TPR < a.N) {
#pragma unroll
                for (int c = 0; c < W; c++) {
                    if (GATED) m[u][c] += g * x[u][c], s[u][c] += vg * (x[u][c] * x[u][c] + v[u][c]) + g * g * v[u][c];
                    else m[u][c] += x[u][c], s[u][c] += v[u][c];
                }
            }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i = i0 + u * TPR;
        if (i >= a.N) break;
        if (!GATED && a.jcb) {
            float q[W];
            load<W>(a.jcb + t * a.N + i, q);
#pragma unroll
            for (int c = 0; c < W; c++) m[u][c] *= q[c], s[u][c] *= q[c] * q[c];
        }
        store<W>(a.mu_y + t * a.N + i, m[u]);
        store<W>(a.var_y + t * a.N + i, s[u]);
    }
}

struct CombineBwdArgs {
    int T, k, N, S;
    const int *pos;
    const float *mu_g, *mu_x, *jcb, *dmu_y, *dvar_y;
    float *dmu_x, *dvar_x, *dmu_g, *dvar_g;
};

// TPR threads per token: the deltas of the slots' rows, and for each slot the sums of x dmu_y and x^2 dvar_y over the features.
// Four slots at a time, so that their rows are fetched together and the token's deltas once.
template <int W, int TPR, bool JCB>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR) combine_bwd_kernel(const CombineBwdArgs a) {
    constexpr int THREADS = TPR == 32 ? 256 : TPR;
    __shared__ float red[TPR / 32][2 * SLOTS];
    const long t = (long)blockIdx.x * (THREADS / TPR) + threadIdx.x / TPR;
    const int u = threadIdx.x % TPR;
    if (TPR == 32 && t >= a.T) return;   // wider: the grid has one CTA per token
    for (int j0 = 0; j0 < a.k; j0 += SLOTS) {
        int p[SLOTS];
        float g[SLOTS], s[2 * SLOTS];
#pragma unroll
        for (int j = 0; j < SLOTS; j++) {
            p[j] = j0 + j < a.k ? slot_row(a.pos, t * a.k + j0 + j, a.S) : -1;
            g[j] = p[j] >= 0 ? __ldg(a.mu_g + t * a.k + j0 + j) : 0.f;
            s[2 * j] = s[2 * j + 1] = 0.f;
        }
        // W = 1: two features at a time, TPR apart
        constexpr int U = W == 4 ? 1 : 2;
        for (int i0 = u * W; i0 < a.N; i0 += TPR * W * U) {
            float dm[U][W], dv[U][W], x[U][SLOTS][W], q[U][SLOTS][W];
#pragma unroll
            for (int h = 0; h < U; h++) {
                const int i = i0 + h * TPR;
                if (i >= a.N) break;
                load<W>(a.dmu_y + t * a.N + i, dm[h]);
                load<W>(a.dvar_y + t * a.N + i, dv[h]);
#pragma unroll
                for (int j = 0; j < SLOTS; j++)
                    if (p[j] >= 0) {
                        load<W>(a.mu_x + (long)p[j] * a.N + i, x[h][j]);
                        if (JCB) load<W>(a.jcb + (long)p[j] * a.N + i, q[h][j]);
                    }
            }
#pragma unroll
            for (int h = 0; h < U; h++) {
                const int i = i0 + h * TPR;
                if (i >= a.N) break;
#pragma unroll
                for (int j = 0; j < SLOTS; j++)
                    if (p[j] >= 0) {
                        float o[W], r[W];
#pragma unroll
                        for (int c = 0; c < W; c++) {
                            const float f = JCB ? g[j] * q[h][j][c] : g[j];
                            s[2 * j] += x[h][j][c] * dm[h][c];
                            s[2 * j + 1] += x[h][j][c] * dv[h][c] * x[h][j][c];
                            o[c] = f * dm[h][c];
                            r[c] = f * dv[h][c] * f;
                        }
                        store<W>(a.dmu_x + (long)p[j] * a.N + i, o);
                        store<W>(a.dvar_x + (long)p[j] * a.N + i, r);
                    }
            }
        }
#pragma unroll
        for (int q = 0; q < 2 * SLOTS; q++) s[q] = warp_sum(s[q]);
        if (TPR > 32) {
            __syncthreads();
            if ((threadIdx.x & 31) == 0)
#pragma unroll
                for (int q = 0; q < 2 * SLOTS; q++) red[threadIdx.x >> 5][q] = s[q];
            __syncthreads();
        }
        if (u < 2 * SLOTS && j0 + u / 2 < a.k) {
            float v = 0.f;
            if (TPR > 32) {
#pragma unroll
                for (int w = 0; w < TPR / 32; w++) v += red[w][u];
            } else {
#pragma unroll
                for (int q = 0; q < 2 * SLOTS; q++)
                    if (q == u) v = s[q];
            }
            ((u & 1) ? a.dvar_g : a.dmu_g)[t * a.k + j0 + u / 2] = v;
        }
    }
}

template <int W, bool GATED>
int combine_fwd_launch(const CombineArgs &a, cudaStream_t st) {
    if (a.N > 512) {
        const long tiles = (a.N + 1023) / 1024;
        if (tiles * a.T >= (1L << 31)) return fail(TAGI_ERR_INVALID_ARGUMENT, "combine: too many tokens times features for one launch");
        combine_fwd_kernel<W, 256, GATED><<<(unsigned)(tiles * a.T), 256, 0, st>>>(a);
    } else if (a.N > 128) {
        combine_fwd_kernel<W, 128, GATED><<<(a.T + 1) / 2, 256, 0, st>>>(a);
    } else if (a.N > 32) {
        combine_fwd_kernel<W, 32, GATED><<<(a.T + 7) / 8, 256, 0, st>>>(a);
    } else {
        combine_fwd_kernel<W, 8, GATED><<<(a.T + 31) / 32, 256, 0, st>>>(a);
    }
    return launched("combine_fwd_kernel launch");
}
template <bool GATED>
int combine_fwd(const CombineArgs &a, cudaStream_t st) {
    if (a.T == 0) return TAGI_OK;
    const bool vec = a.N % 4 == 0 && all16({a.mu_x, a.var_x, a.jcb, a.mu_y, a.var_y});
    return vec ? combine_fwd_launch<4, GATED>(a, st) : combine_fwd_launch<1, GATED>(a, st);
}

}  // namespace
}  // namespace tagi

using namespace tagi;

#define TAGI_PTR(p) TAGI_REQUIRE((p) != nullptr && aligned4(p), #p " is null or not 4-byte aligned")
#define TAGI_PTR_IF(cond, p) TAGI_REQUIRE(!(cond) || ((p) != nullptr && aligned4(p)), #p " is null or not 4-byte aligned")

extern "C" {

int tagi_ln_fwd(int R, int n, int has_bias, float eps, const float *mu_w, const float *var_w, const float *mu_b,
                const float *var_b, const float *mu_a, const float *var_a, float *mu_row, float *var_row, float *mu_z,
                float *var_z, void *stream) {
    TAGI_REQUIRE(R >= 0 && n >= 2, "rows must not be negative, features must be at least 2 (the variance divides by n - 1)");
    TAGI_REQUIRE(R <= MAX_ROWS && n <= MAX_FEATURES, "more than 2^30 rows or 2^24 features");
    TAGI_REQUIRE(eps >= 0.f, "eps must not be negative");
    TAGI_PTR(mu_w);
    TAGI_PTR(var_w);
    TAGI_PTR_IF(has_bias, mu_b);
    TAGI_PTR_IF(has_bias, var_b);
    if (R == 0) return TAGI_OK;
    TAGI_PTR(mu_a);
    TAGI_PTR(var_a);
    TAGI_PTR(mu_row);
    TAGI_PTR(var_row);
    TAGI_PTR(mu_z);
    TAGI_PTR(var_z);
    const LnArgs a{R, n, eps, mu_w, var_w, has_bias ? mu_b : nullptr, has_bias ? var_b : nullptr, mu_a, var_a, mu_row,
                   var_row, mu_z, var_z};
    const bool vec = n % 4 == 0 && all16({mu_w, var_w, a.mu_b, a.var_b, mu_a, var_a, mu_z, var_z});
    return vec ? ln_fwd_launch<4>(a, static_cast<cudaStream_t>(stream)) : ln_fwd_launch<1>(a, static_cast<cudaStream_t>(stream));
}

size_t tagi_ln_bwd_workspace_bytes(int R, int n) {
    if (R < 0 || n < 2 || R > MAX_ROWS || n > MAX_FEATURES) return 0;
    const int chunks = ln_bwd_chunks(R, n);
    return chunks <= 1 ? 0 : (size_t)chunks * 4 * n * sizeof(float);
}

int tagi_ln_bwd(int R, int n, int has_bias, int state_update, float eps, const float *mu_w, const float *var_w,
                const float *var_b, const float *mu_a, const float *jcb, const float *mu_row, const float *var_row,
                const float *dmu_o, const float *dvar_o, float *dmu, float *dvar, float *dmu_w, float *dvar_w, float *dmu_b,
                float *dvar_b, void *workspace, size_t workspace_bytes, void *stream) {
    TAGI_REQUIRE(R >= 0 && n >= 2, "rows must not be negative, features must be at least 2");
    TAGI_REQUIRE(R <= MAX_ROWS && n <= MAX_FEATURES, "more than 2^30 rows or 2^24 features");
    TAGI_REQUIRE(eps >= 0.f, "eps must not be negative");
    TAGI_PTR(mu_w);
    TAGI_PTR(var_w);
    TAGI_PTR(dmu_w);
    TAGI_PTR(dvar_w);
    TAGI_PTR_IF(has_bias, var_b);
    TAGI_PTR_IF(has_bias, dmu_b);
    TAGI_PTR_IF(has_bias, dvar_b);
    TAGI_PTR_IF(R > 0, mu_a);
    TAGI_PTR_IF(R > 0, mu_row);
    TAGI_PTR_IF(R > 0, var_row);
    TAGI_PTR_IF(R > 0, dmu_o);
    TAGI_PTR_IF(R > 0, dvar_o);
    TAGI_PTR_IF(R > 0 && state_update, dmu);
    TAGI_PTR_IF(R > 0 && state_update, dvar);
    TAGI_REQUIRE(jcb == nullptr || aligned4(jcb), "jcb is not 4-byte aligned");
    const size_t need = tagi_ln_bwd_workspace_bytes(R, n);
    TAGI_REQUIRE(need == 0 || (workspace != nullptr && aligned16(workspace) && workspace_bytes >= need),
                 "workspace is null, not 16-byte aligned or smaller than tagi_ln_bwd_workspace_bytes");
    LnBwdArgs a{R, n, ln_bwd_chunk(R, n), eps, mu_w, var_w, has_bias ? var_b : nullptr, mu_a, jcb, mu_row, var_row, dmu_o,
                dvar_o, state_update ? dmu : nullptr, state_update ? dvar : nullptr, dmu_w, dvar_w, dmu_b, dvar_b,
                need ? static_cast<float *>(workspace) : nullptr};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int chunks = ln_bwd_chunks(R, n);
    const bool vec = n % 4 == 0 && all16({mu_w, mu_a, jcb, dmu_o, dvar_o, a.dmu, a.dvar});
    const int per = LN_BWD_THREADS * (vec || n >= 384 ? 4 : 1);
    const dim3 grid((n + per - 1) / per, chunks > 1 ? chunks : 1);   // no rows: one empty chunk writes the zeros
    if (vec) ln_bwd_kernel<4, 1><<<grid, LN_BWD_THREADS, 0, st>>>(a);
    else if (n >= 384) ln_bwd_kernel<1, 4><<<grid, LN_BWD_THREADS, 0, st>>>(a);
    else ln_bwd_kernel<1, 1><<<grid, LN_BWD_THREADS, 0, st>>>(a);
    int rc = launched("ln_bwd_kernel launch");
    if (rc != TAGI_OK || chunks <= 1) return rc;
    ln_bwd_final_kernel<<<dim3((n + 31) / 32, has_bias ? 4 : 2), FINAL_GROUPS * 32, 0, st>>>(a, chunks);
    return launched("ln_bwd_final_kernel launch");
}

static int check_slots(const char *who, int T, int k, int N, int S, const int *pos) {
    if (T < 0 || S < 0 || k < 1 || N < 1)
        return fail(TAGI_ERR_INVALID_ARGUMENT, std::string(who) + ": sizes must be positive (tokens and rows may be zero)");
    if (T > MAX_ROWS || N > MAX_FEATURES) return fail(TAGI_ERR_INVALID_ARGUMENT, std::string(who) + ": more than 2^30 tokens or 2^24 features");
    if ((long)T * k >= (1L << 31)) return fail(TAGI_ERR_INVALID_ARGUMENT, std::string(who) + ": more than 2^31 slots");
    if (T > 0 && (pos == nullptr || !aligned4(pos)))
        return fail(TAGI_ERR_INVALID_ARGUMENT, std::string(who) + ": pos is null or not 4-byte aligned");
    return TAGI_OK;
}

int tagi_combine_fwd(int T, int k, int N, int S, const int *pos, const float *mu_g, const float *var_g, const float *mu_x,
                     const float *var_x, float *mu_y, float *var_y, void *stream) {
    int rc = check_slots(__func__, T, k, N, S, pos);
    if (rc != TAGI_OK || T == 0) return rc;
    TAGI_PTR(mu_g);
    TAGI_PTR(var_g);
    TAGI_PTR_IF(S > 0, mu_x);
    TAGI_PTR_IF(S > 0, var_x);
    TAGI_PTR(mu_y);
    TAGI_PTR(var_y);
    return combine_fwd<true>(CombineArgs{T, k, N, S, pos, mu_g, var_g, mu_x, var_x, nullptr, mu_y, var_y},
                             static_cast<cudaStream_t>(stream));
}

int tagi_dispatch_bwd(int T, int k, int N, int S, const int *pos, const float *jcb, const float *dmu_x, const float *dvar_x,
                      float *dmu_a, float *dvar_a, void *stream) {
    int rc = check_slots(__func__, T, k, N, S, pos);
    if (rc != TAGI_OK || T == 0) return rc;
    TAGI_PTR_IF(S > 0, dmu_x);
    TAGI_PTR_IF(S > 0, dvar_x);
    TAGI_PTR(dmu_a);
    TAGI_PTR(dvar_a);
    TAGI_REQUIRE(jcb == nullptr || aligned4(jcb), "jcb is not 4-byte aligned");
    return combine_fwd<false>(CombineArgs{T, k, N, S, pos, nullptr, nullptr, dmu_x, dvar_x, jcb, dmu_a, dvar_a},
                              static_cast<cudaStream_t>(stream));
}

int tagi_combine_bwd(int T, int k, int N, int S, const int *pos, const float *mu_g, const float *mu_x, const float *jcb,
                     const float *dmu_y, const float *dvar_y, float *dmu_x, float *dvar_x, float *dmu_g, float *dvar_g,
                     void *stream) {
    int rc = check_slots(__func__, T, k, N, S, pos);
    if (rc != TAGI_OK || T == 0) return rc;
    TAGI_PTR(mu_g);
    TAGI_PTR_IF(S > 0, mu_x);
    TAGI_PTR(dmu_y);
    TAGI_PTR(dvar_y);
    TAGI_PTR_IF(S > 0, dmu_x);
    TAGI_PTR_IF(S > 0, dvar_x);
    TAGI_PTR(dmu_g);
    TAGI_PTR(dvar_g);
    TAGI_REQUIRE(jcb == nullptr || aligned4(jcb), "jcb is not 4-byte aligned");
    const CombineBwdArgs a{T, k, N, S, pos, mu_g, mu_x, jcb, dmu_y, dvar_y, dmu_x, dvar_x, dmu_g, dvar_g};
    // A warp per token up to two of its strides, else a CTA of 128: 8192 tokens, four rows of 1024: 79 us (a warp 85 us, a CTA
    // of 256 threads 85 us); 16384 tokens, two rows of 2048: 184 us (197 and 195 us).
    const bool vec = N % 4 == 0 && all16({mu_x, jcb, dmu_y, dvar_y, dmu_x, dvar_x});
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto start = [&](auto with) {
        constexpr bool J = decltype(with)::value;
        if (vec && N > 256) combine_bwd_kernel<4, 128, J><<<T, 128, 0, st>>>(a);
        else if (vec) combine_bwd_kernel<4, 32, J><<<(T + 7) / 8, 256, 0, st>>>(a);
        else if (N > 128) combine_bwd_kernel<1, 128, J><<<T, 128, 0, st>>>(a);
        else combine_bwd_kernel<1, 32, J><<<(T + 7) / 8, 256, 0, st>>>(a);
    };
    if (jcb) start(std::true_type());
    else start(std::false_type());
    return launched("combine_bwd_kernel launch");
}

}  // extern "C"
