// Linear layers grouped by expert, experts with few rows: every weight is read once and met by all rows of its expert, on
// the FP32 pipe. These passes are bound by HBM (8, 4 and 12 bytes a weight in the forward, state and parameter pass) until
// the rows' multiplications (3, 2 and 2 a weight and row) take longer, at about 14, 11 and 33 rows. Experts with more than
// `few` rows are left to the tensor-core kernels, which in turn leave these alone; the offsets are device data, so all are
// launched unless the number of rows in all rules one out.
//
// Forward and state pass: a CTA computes 64 output columns of all the expert's rows. The weights come in slabs of 32
// contraction steps through a ring of stages filled with cp.async, so that the bytes in flight cost no registers (two CTAs of
// an SM keep about 100 KB on their way). Where there are too few tiles for that, a cluster of up to eight CTAs cuts the
// contraction of a tile, and their sums are added through distributed shared memory in the order of the CTAs. Eight warps share a slab, four steps each; a
// thread multiplies its two columns with all rows, whose entries all lanes read at the same address. The warps' sums are
// added in a fixed order at the end.
#include "tagi_grouped.h"

namespace tagi {
namespace {

constexpr int OUT = 64, SLAB = 32, WARPS = 8, THREADS = WARPS * 32, ROWS = FEW_ROWS;
static_assert(SLAB == 4 * WARPS, "a warp takes four steps of a slab");
constexpr int PITCH = SLAB + 4;                          // floats of a weight row in shared memory: no bank conflicts
constexpr int FWD_WEIGHTS = 2 * OUT * PITCH, STATE_WEIGHTS = SLAB * OUT;
__host__ __device__ constexpr int stages(int pass) { return pass == FWD ? 4 : 8; }   // a slab of both is 18 KiB, of means 8

__device__ __forceinline__ uint32_t smem_at(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// Four floats to shared memory, of which the first `valid` (any number, also none or more than four) exist; zeros else.
template <bool VEC>
__device__ __forceinline__ void copy4(float *dst, const float *src, int valid) {
    const uint32_t d = smem_at(dst);
    if (VEC) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(valid > 0 ? 16 : 0) : "memory");
    } else {
#pragma unroll
        for (int c = 0; c < 4; c++)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d + c * 4), "l"(src + (c < valid ? c : 0)), "r"(c < valid ? 4 : 0)
                         : "memory");
    }
}
__device__ __forceinline__ float4 at4(const float *p) { return *reinterpret_cast<const float4 *>(p); }

// Two contraction steps of a sum in one register pair: two multiply-adds are one instruction.
typedef unsigned long long Pair;
__device__ __forceinline__ Pair pair_of(float a, float b) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// float at the same place in the shared memory of CTA `cta` of the cluster
__device__ __forceinline__ float remote(const float *p, int cta) {
    float v;
    asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %1, %2;\n\tld.shared::cluster.f32 %0, [r];\n\t}" : "=f"(v) : "r"(smem_at(p)), "r"(cta) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float sum_of(Pair p) {
    float a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
    return a + b;
}

// smem: a ring of stages of weights and rows, used again for the warps' sums.
template <int PASS, bool VEC>
__device__ __forceinline__ void few_rows_pass(const GroupedArgs &a, int e, int r0, int rows, float *smem) {
    constexpr int WEIGHTS = PASS == FWD ? FWD_WEIGHTS : STATE_WEIGHTS, STAGE = WEIGHTS + 2 * ROWS * SLAB, STAGES = stages(PASS);
    const int tid = threadIdx.x, lane = tid & 31, q = tid >> 5;   // q: the warp, and its four steps of a slab
    const int o0 = blockIdx.x * OUT, outs = PASS == FWD ? a.N : a.K, depth = PASS == FWD ? a.K : a.N;
    const size_t wbase = (size_t)e * a.N * a.K;

    // this thread's copy of the rows: quad tid & 7 of row (tid >> 3) % ROWS, means first
    static_assert(2 * ROWS * 8 <= THREADS, "one copy a thread");
    const int mine = tid < 2 * ROWS * 8 && (tid >> 3) % ROWS < rows ? r0 + (tid >> 3) % ROWS : -1;
    const int row = mine < 0 ? -1 : PASS == FWD ? input_row(a, mine) : mine;
    auto fetch = [&](int slab, int last) {
        const int k0 = slab * SLAB;
        float *s = smem + (slab % STAGES) * STAGE;
        if (slab < last) {
            if (PASS == FWD) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int c = tid + (i & 1) * THREADS, n = c >> 3, k = k0 + (c & 7) * 4;
                    copy4<VEC>(s + (i >> 1) * OUT * PITCH + n * PITCH + (c & 7) * 4,
                               (i < 2 ? a.mu_w : a.var_w) + (o0 + n < a.N ? wbase + (size_t)(o0 + n) * a.K + (k < a.K ? k : 0) : 0),
                               o0 + n < a.N ? a.K - k : 0);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int c = tid + i * THREADS, n = k0 + (c >> 4), k = o0 + (c & 15) * 4;
                    copy4<VEC>(s + (c >> 4) * OUT + (c & 15) * 4, a.mu_w + (n < a.N ? wbase + (size_t)n * a.K + (k < a.K ? k : 0) : 0),
                               n < a.N ? a.K - k : 0);
                }
            }
            if (tid < 2 * ROWS * 8) {
                const int k = k0 + (tid & 7) * 4;
                copy4<VEC>(s + WEIGHTS + tid * 4, (tid < ROWS * 8 ? a.a0 : a.a1) + (row >= 0 && k < depth ? (size_t)row * depth + k : 0),
                           row >= 0 ? depth - k : 0);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    Pair z[2][ROWS], vz[2][ROWS];
#pragma unroll
    for (int t = 0; t < ROWS; t++) z[0][t] = z[1][t] = vz[0][t] = vz[1][t] = 0;
    // this CTA's slabs of the cluster's
    const int parts = gridDim.z, all = (depth + SLAB - 1) / SLAB, first = (int)((long)all * blockIdx.z / parts),
              last = (int)((long)all * (blockIdx.z + 1) / parts);
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++) fetch(first + s, last);
    for (int it = first; it < last; it++) {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncthreads();   // slab `it` is there for all, and nobody reads the stage that is filled next any more
        fetch(it + STAGES - 1, last);
        const float *w = smem + (it % STAGES) * STAGE, *x = w + WEIGHTS, *y = x + ROWS * SLAB;
        {
            Pair wm[2][2], wq[2][2], wv[2][2];   // the thread's two columns at four steps: means, their squares, variances
#pragma unroll
            for (int f = 0; f < 2; f++) {
                if (PASS == FWD) {
                    const float4 m = at4(w + (f * 32 + lane) * PITCH + q * 4), v = at4(w + OUT * PITCH + (f * 32 + lane) * PITCH + q * 4);
                    wm[f][0] = pair_of(m.x, m.y), wm[f][1] = pair_of(m.z, m.w);
                    wv[f][0] = pair_of(v.x, v.y), wv[f][1] = pair_of(v.z, v.w);
                } else {
                    const float *p = w + q * 4 * OUT + f * 32 + lane;
                    wm[f][0] = pair_of(p[0], p[OUT]), wm[f][1] = pair_of(p[2 * OUT], p[3 * OUT]);
                }
                wq[f][0] = mul2(wm[f][0], wm[f][0]), wq[f][1] = mul2(wm[f][1], wm[f][1]);
            }
#pragma unroll
            for (int t = 0; t < ROWS; t++)
                if (t < rows) {
                    const float4 xt = at4(x + t * SLAB + q * 4), yt = at4(y + t * SLAB + q * 4);
                    const Pair xs[2] = {pair_of(xt.x, xt.y), pair_of(xt.z, xt.w)}, ys[2] = {pair_of(yt.x, yt.y), pair_of(yt.z, yt.w)};
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const Pair second = PASS == FWD ? fma2(xs[c], xs[c], ys[c]) : 0;
#pragma unroll
                        for (int f = 0; f < 2; f++) {
                            z[f][t] = fma2(xs[c], wm[f][c], z[f][t]);
                            vz[f][t] = fma2(ys[c], wq[f][c], vz[f][t]);
                            if (PASS == FWD) vz[f][t] = fma2(second, wv[f][c], vz[f][t]);
                        }
                    }
                }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    // red[warp][row][kind][column]
    float *red = smem;
#pragma unroll
    for (int t = 0; t < ROWS; t++)
#pragma unroll
        for (int f = 0; f < 2; f++) {
            const int at = ((q * ROWS + t) * 2) * OUT + f * 32 + lane;
            red[at] = sum_of(z[f][t]);
            red[at + OUT] = sum_of(vz[f][t]);
        }
    if (parts > 1) cluster_sync();
    else __syncthreads();
    for (int i = blockIdx.z * THREADS + tid; i < rows * 2 * OUT; i += parts * THREADS) {
        float s = 0.f;
        for (int c = 0; c < parts; c++)
#pragma unroll
            for (int p = 0; p < WARPS; p++) s += parts > 1 ? remote(red + p * ROWS * 2 * OUT + i, c) : red[p * ROWS * 2 * OUT + i];
        const int c = o0 + (i & (OUT - 1)), r = i / (2 * OUT);
        const bool var = (i / OUT) & 1;
        if (c >= outs) continue;
        const size_t o = (size_t)(r0 + r) * outs + c;
        if (PASS == FWD) {
            if (a.mu_b) s += __ldg((var ? a.var_b : a.mu_b) + (size_t)e * a.N + c);
        } else if (a.jcb) {
            const float j = __ldg(a.jcb + o);
            s = var ? s * j * j : s * j;
        }
        (var ? a.o1 : a.o0)[o] = s;
    }
    if (parts > 1) cluster_sync();   // nobody leaves while its sums are read
}

template <int PASS, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) grouped_few_kernel(const GroupedArgs a) {
    extern __shared__ __align__(16) float smem[];
    int r0, r1;
    expert_rows(a, blockIdx.y, r0, r1);
    if (r1 > r0 && r1 - r0 <= a.few) few_rows_pass<PASS, VEC>(a, blockIdx.y, r0, r1 - r0, smem);   // the same in the whole cluster
}

// -------------------------------------------------------------------------------------------------------- parameters
// A warp computes PARAM_N output features x 32 lanes of W input features; a CTA stacks 8 warps along the output features. The
// prior variances are fetched before the rows are added up; the deltas come from shared memory, at one address for all lanes.
constexpr int PARAM_N = 8, PARAM_OUT = WARPS * PARAM_N;

template <int W>
__device__ __forceinline__ void load(const float *p, float (&v)[W]) {
    if (W == 4) {
        const float4 t = __ldg(reinterpret_cast<const float4 *>(p));
        v[0] = t.x, v[1 % W] = t.y, v[2 % W] = t.z, v[3 % W] = t.w;
    } else {
        v[0] = __ldg(p);
    }
}

// weights pass by once: they are kept out of L1, where the rows are wanted
template <int W>
__device__ __forceinline__ void load_once(const float *p, float (&v)[W]) {
    if (W == 4)
        asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v[0]), "=f"(v[1 % W]), "=f"(v[2 % W]), "=f"(v[3 % W])
                     : "l"(p));
    else
        asm volatile("ld.global.nc.L1::no_allocate.f32 %0, [%1];" : "=f"(v[0]) : "l"(p));
}

template <int W>
__global__ void __launch_bounds__(THREADS, 2) grouped_few_param_kernel(const GroupedArgs a) {
    __shared__ __align__(16) float delta[FEW_PARAM_ROWS][2][PARAM_OUT];
    __shared__ int input[FEW_PARAM_ROWS];
    const int e = blockIdx.z;
    int r0, r1;
    expert_rows(a, e, r0, r1);
    const int rows = r1 - r0;
    if (rows > a.few) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, block_n = blockIdx.y * PARAM_OUT, n0 = block_n + warp * PARAM_N;
    const int k = (blockIdx.x * 32 + lane) * W;
    const bool live = k < a.K;
    float d[PARAM_N][W], v[PARAM_N][W], s[PARAM_N][W];
    const size_t o = ((size_t)e * a.N + n0) * a.K + k;
#pragma unroll
    for (int i = 0; i < PARAM_N; i++) {
#pragma unroll
        for (int c = 0; c < W; c++) d[i][c] = v[i][c] = s[i][c] = 0.f;
        if (live && rows > 0 && n0 + i < a.N) load_once<W>(a.var_w + o + (size_t)i * a.K, s[i]);
    }
    for (int i = threadIdx.x; i < rows * 2 * PARAM_OUT; i += THREADS) {
        const int n = block_n + i % PARAM_OUT, r = i / (2 * PARAM_OUT);
        delta[r][(i / PARAM_OUT) & 1][i % PARAM_OUT] = n < a.N ? __ldg(((i / PARAM_OUT) & 1 ? a.a1 : a.a0) + (size_t)(r0 + r) * a.N + n) : 0.f;
    }
    for (int r = threadIdx.x; r < rows; r += THREADS) input[r] = input_row(a, r0 + r);
    __syncthreads();
    if (a.var_b && blockIdx.x == 0 && threadIdx.x < 2 * PARAM_OUT) {
        const int kind = threadIdx.x / PARAM_OUT, n = block_n + threadIdx.x % PARAM_OUT;
        if (n < a.N) {
            float t = 0.f;
            for (int r = 0; r < rows; r++) t += delta[r][kind][threadIdx.x % PARAM_OUT];
            const float vb = __ldg(a.var_b + (size_t)e * a.N + n);
            (kind ? a.ob1 : a.ob0)[(size_t)e * a.N + n] = kind ? vb * vb * t : vb * t;
        }
    }
    if (!live) return;
#pragma unroll 2
    for (int r = 0; r < rows; r++) {
        const int row = input[r];
        float x[W], q[W];
#pragma unroll
        for (int c = 0; c < W; c++) x[c] = 0.f;
        if (row >= 0) load<W>(a.x + (size_t)row * a.K + k, x);
#pragma unroll
        for (int c = 0; c < W; c++) q[c] = x[c] * x[c];
#pragma unroll
        for (int h = 0; h < PARAM_N; h += 4) {
            const float4 m = at4(&delta[r][0][warp * PARAM_N + h]), u = at4(&delta[r][1][warp * PARAM_N + h]);
            const float dm[4] = {m.x, m.y, m.z, m.w}, dv[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int c = 0; c < W; c++) d[h + i][c] = fmaf(dm[i], x[c], d[h + i][c]), v[h + i][c] = fmaf(dv[i], q[c], v[h + i][c]);
        }
    }
#pragma unroll
    for (int i = 0; i < PARAM_N; i++) {
        if (n0 + i >= a.N) break;
#pragma unroll
        for (int c = 0; c < W; c++) d[i][c] *= s[i][c], v[i][c] *= s[i][c] * s[i][c];
        float *p = a.o0 + o + (size_t)i * a.K, *u = a.o1 + o + (size_t)i * a.K;
        if (W == 4) {
            __stcs(reinterpret_cast<float4 *>(p), make_float4(d[i][0], d[i][1 % W], d[i][2 % W], d[i][3 % W]));
            __stcs(reinterpret_cast<float4 *>(u), make_float4(v[i][0], v[i][1 % W], v[i][2 % W], v[i][3 % W]));
        } else {
            __stcs(p, d[i][0]);
            __stcs(u, v[i][0]);
        }
    }
}

template <int PASS, bool VEC>
int launch_few(const GroupedArgs &a, cudaStream_t st) {
    constexpr size_t ring = stages(PASS) * ((PASS == FWD ? FWD_WEIGHTS : STATE_WEIGHTS) + 2 * ROWS * SLAB), sums = WARPS * ROWS * 2 * OUT;
    constexpr size_t smem = (ring > sums ? ring : sums) * sizeof(float);
    // CTAs that have work, at most: with fewer than two for an SM, clusters cut the contraction, into no less than 256 steps
    const int tiles = ((PASS == FWD ? a.N : a.K) + OUT - 1) / OUT, depth = PASS == FWD ? a.K : a.N;
    const long ctas = (long)tiles * (a.E < a.S ? a.E : a.S);
    int parts = 1;
    while (parts < 8 && ctas * parts < 2 * 148 && depth >= 512 * parts) parts *= 2;
    auto k = grouped_few_kernel<PASS, VEC>;
    TAGI_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles, a.E, parts);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = parts;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    TAGI_CUDA(cudaLaunchKernelEx(&cfg, k, a));
    return TAGI_OK;
}

template <int PASS>
int launch(const GroupedArgs &a, cudaStream_t st) {
    return grouped_aligned(PASS, a) ? launch_few<PASS, true>(a, st) : launch_few<PASS, false>(a, st);
}

}  // namespace

int grouped_few(int pass, const GroupedArgs &a, cudaStream_t st) {
    if (pass == FWD) return launch<FWD>(a, st);
    if (pass == STATE) return launch<STATE>(a, st);
    const bool vec = a.K % 4 == 0 && aligned16(a.var_w) && aligned16(a.x) && aligned16(a.o0) && aligned16(a.o1);
    const int per = 32 * (vec ? 4 : 1);
    const dim3 grid((a.K + per - 1) / per, (a.N + PARAM_OUT - 1) / PARAM_OUT, a.E);
    if (vec) grouped_few_param_kernel<4><<<grid, THREADS, 0, st>>>(a);
    else grouped_few_param_kernel<1><<<grid, THREADS, 0, st>>>(a);
    TAGI_CUDA(cudaGetLastError());
    return TAGI_OK;
}

}  // namespace tagi
