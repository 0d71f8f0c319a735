// Linear layers grouped by expert, experts with few rows: every weight is read once and met by all rows of its expert, on
// the FP32 pipe. These passes are bound by HBM (8, 4 and 12 bytes a weight in the forward, state and parameter pass) until
// the rows' multiplications (3, 2 and 2 a weight and row) take longer, at about 14, 11 and 33 rows. Experts with more than
// `few` rows are left to the tensor-core kernels, which in turn leave these alone; the offsets are device data, so all are
// launched unless the number of rows in all rules one out.
//
// Forward and state pass: a CTA computes 64 output columns of all the expert's rows. The weights come in slabs of 32
// contraction steps through a ring of stages filled with cp.async, so that the bytes in flight cost no registers (two CTAs of
// an SM keep about 100 KB on their way). Where there are too few tiles for that, a cluster of up to eight CTAs cuts the
// contraction of a tile, and their sums are added through distributed shared memory in the order of the CTAs. Eight warps share
// a slab, four steps each; a thread multiplies its two columns with all rows, whose entries all lanes read at the same address.
// The warps' sums are added in a fixed order at the end.
#include "tagi_grouped.h"

namespace tagi {
namespace {

constexpr int OUT = 64, SLAB = 32, WARPS = 8, THREADS = WARPS * 32, ROWS = FEW_ROWS;
static_assert(SLAB == 4 * WARPS, "a warp takes four steps of a slab");
constexpr int PITCH = SLAB + 4;                          // floats of a weight row in shared memory: no bank conflicts
constexpr int FWD_WEIGHTS = 2 * OUT * PITCH;
// Rows that do not begin at multiples of 16 bytes are copied in the 16-byte groups of memory all the same, one more of them,
// and begin up to three floats behind their place in shared memory. One row of two experts of 4095 x 4095, forward: 70 us,
// with 4-byte copies 94 us; of 4096 x 4096 57 us.
__host__ __device__ constexpr int state_pitch(bool vec) { return vec ? OUT : OUT + 4; }
__host__ __device__ constexpr int weights(int pass, bool vec) { return pass == FWD ? FWD_WEIGHTS : SLAB * state_pitch(vec); }
__host__ __device__ constexpr int stages(int pass) { return pass == FWD ? 4 : 8; }   // a slab of both is 18 KiB, of means 8

__device__ __forceinline__ float4 at4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
// four floats from p + shift on, p aligned
__device__ __forceinline__ float4 at4(const float *p, int shift) {
    const float4 a = at4(p), b = at4(p + 4);
    const bool one = shift & 1, two = shift & 2;
    const float x = one ? a.y : a.x, y = one ? a.z : a.y, z = one ? a.w : a.z, w = one ? b.x : a.w, u = one ? b.y : b.x, v = one ? b.z : b.y;
    return make_float4(two ? z : x, two ? w : y, two ? u : z, two ? v : w);
}

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
    asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %1, %2;\n\tld.shared::cluster.f32 %0, [r];\n\t}"
                 : "=f"(v)
                 : "r"(smem_at(p)), "r"(cta)
                 : "memory");
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
    constexpr int WEIGHTS = weights(PASS, VEC), SP = state_pitch(VEC), STAGE = WEIGHTS + 2 * ROWS * SLAB, STAGES = stages(PASS);
    const int tid = threadIdx.x, lane = tid & 31, q = tid >> 5;   // q: the warp, and its four steps of a slab
    const int o0 = blockIdx.x * OUT, outs = PASS == FWD ? a.N : a.K, depth = PASS == FWD ? a.K : a.N;
    const size_t wbase = (size_t)e * a.N * a.K;

    // this CTA's slabs of the cluster's
    const int parts = gridDim.z, all = (depth + SLAB - 1) / SLAB, first = (int)((long)all * blockIdx.z / parts),
              last = (int)((long)all * (blockIdx.z + 1) / parts);

    // What this thread copies of a slab, as addresses that move on by a slab each time (working them out anew took more
    // instructions than all else). Weights: forward, group tid & 7 of lines n and n + 32 of both tensors; state, group tid & 15
    // of lines n and n + 16. Lines that are so far apart begin equally far from a multiple of 16 bytes. Where that is not zero
    // a line has one more group, `more`.
    constexpr int FAR = PASS == FWD ? 32 : 16, GROUPS = PASS == FWD ? 8 : 16;
    const int n = tid / GROUPS, g = (tid % GROUPS) * 4;
    const size_t far = (size_t)FAR * a.K, move = PASS == FWD ? SLAB : (size_t)SLAB * a.K;
    const float *pm = a.mu_w + wbase + (PASS == FWD ? (size_t)(o0 + n) * a.K + first * SLAB : (size_t)(first * SLAB + n) * a.K + o0), *pv = nullptr;
    int at = PASS == FWD ? first * SLAB : o0;   // place of the slab's first column in its line
    const int sm = VEC ? 0 : shift_of(pm);
    int sv = 0;
    pm += g - sm;
    if (PASS == FWD) {
        pv = a.var_w + wbase + (size_t)(o0 + n) * a.K + first * SLAB;
        sv = VEC ? 0 : shift_of(pv);
        pv += g - sv;
    }
    const int extra = PASS == FWD ? tid & (OUT - 1) : tid;   // the line whose last group this thread copies: forward, of means, then of variances
    const bool has_extra = !VEC && (PASS == FWD ? tid < 2 * OUT && o0 + extra < a.N : tid < SLAB);
    const float *more = nullptr;
    int se = 0;
    if (!VEC) {
        more = (PASS == FWD && tid >= OUT ? a.var_w : a.mu_w) + wbase +
               (PASS == FWD ? (size_t)(o0 + extra) * a.K + first * SLAB : (size_t)(first * SLAB + extra) * a.K + o0);
        se = shift_of(more);
        more += GROUPS * 4 - se;
    }
    const bool tensor_begins = !VEC && blockIdx.y == 0 && n == 0 && g == 0 && o0 == 0 && first == 0;   // its first group may begin before it

    // and of the rows: four entries (VEC: threads of means, then of variances), or one of both
    const int t = VEC ? (tid >> 3) % ROWS : tid >> 5, tk = VEC ? (tid & 7) * 4 : lane;
    const bool mine = t < rows && (!VEC || tid < 2 * ROWS * 8);
    const int row = !mine ? -1 : PASS == FWD ? input_row(a, r0 + t) : r0 + t;
    const size_t row_at = (size_t)max(row, 0) * depth + first * SLAB + tk;
    const float *px = (VEC && tid >= ROWS * 8 ? a.a1 : a.a0) + row_at, *py = a.a1 + row_at;
    auto fetch = [&](int slab) {
        const int k0 = slab * SLAB;
        float *s = smem + (slab % STAGES) * STAGE;
        if (slab < last) {
            if (PASS == FWD) {
                const bool in = o0 + n < a.N, in_far = o0 + n + FAR < a.N;
                const int lm = a.K - at + sm - g, lv = a.K - at + sv - g;
                float *d = s + n * PITCH + g;
                if (in) {
                    if (tensor_begins && slab == 0 && (sm | sv) != 0) {
                        copy_first_group(d, pm, sm, lm);
                        copy_first_group(d + OUT * PITCH, pv, sv, lv);
                    } else {
                        copy_group(d, pm, lm);
                        copy_group(d + OUT * PITCH, pv, lv);
                    }
                }
                if (in_far) {
                    copy_group(d + FAR * PITCH, pm + far, lm);
                    copy_group(d + (OUT + FAR) * PITCH, pv + far, lv);
                }
                if (has_extra) copy_group(s + (tid >> 6) * OUT * PITCH + extra * PITCH + GROUPS * 4, more, a.K - at + se - GROUPS * 4);
                at += SLAB, pv += move;
            } else {
                const int lm = a.K - at + sm - g, le = a.K - at + se - GROUPS * 4;   // lines behind the last: zeros
                float *d = s + n * SP + g;
                if (tensor_begins && slab == 0 && sm != 0) copy_first_group(d, pm, sm, lm);
                else copy_group(d, pm, k0 + n < a.N ? lm : 0);
                copy_group(d + FAR * SP, pm + far, k0 + n + FAR < a.N ? lm : 0);
                if (has_extra) copy_group(s + extra * SP + GROUPS * 4, more, k0 + extra < a.N ? le : 0);
            }
            pm += move;
            if (!VEC) more += move;
            if (mine) {
                const bool in = row >= 0 && k0 + tk < depth;
                if (VEC) {
                    copy_group(s + WEIGHTS + tid * 4, px, in ? 4 : 0);
                } else {
                    copy_float(s + WEIGHTS + t * SLAB + lane, px, in);
                    copy_float(s + WEIGHTS + (ROWS + t) * SLAB + lane, py, in);
                    py += SLAB;
                }
                px += SLAB;
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // shifts of what this thread reads, the same in all slabs (32 floats apart, or 32 rows): forward pass, its two columns' means
    // and variances; state pass, its four steps
    int shift[2][2] = {};
    if (!VEC) {
#pragma unroll
        for (int f = 0; f < 2; f++)
#pragma unroll
            for (int v = 0; v < 2; v++)
                shift[f][v] = PASS == FWD ? shift_of((v ? a.var_w : a.mu_w) + wbase + (size_t)(o0 + f * 32 + lane) * a.K)
                                          : shift_of(a.mu_w + wbase + (size_t)(q * 4 + f * 2 + v) * a.K);
    }
    Pair z[2][ROWS], vz[2][ROWS];
#pragma unroll
    for (int t = 0; t < ROWS; t++) z[0][t] = z[1][t] = vz[0][t] = vz[1][t] = 0;
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++) fetch(first + s);
    for (int it = first; it < last; it++) {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncthreads();   // slab `it` is there for all, and nobody reads the stage that is filled next any more
        fetch(it + STAGES - 1);
        const float *w = smem + (it % STAGES) * STAGE, *x = w + WEIGHTS, *y = x + ROWS * SLAB;
        {
            Pair wm[2][2], wq[2][2], wv[2][2];   // the thread's two columns at four steps: means, their squares, variances
#pragma unroll
            for (int f = 0; f < 2; f++) {
                if (PASS == FWD) {
                    const float *p = w + (f * 32 + lane) * PITCH + q * 4;
                    const float4 m = VEC ? at4(p) : at4(p, shift[f][0]), v = VEC ? at4(p + OUT * PITCH) : at4(p + OUT * PITCH, shift[f][1]);
                    wm[f][0] = pair_of(m.x, m.y), wm[f][1] = pair_of(m.z, m.w);
                    wv[f][0] = pair_of(v.x, v.y), wv[f][1] = pair_of(v.z, v.w);
                } else {
                    const float *p = w + q * 4 * SP + f * 32 + lane;
                    wm[f][0] = pair_of(p[shift[0][0]], p[SP + shift[0][1]]), wm[f][1] = pair_of(p[2 * SP + shift[1][0]], p[3 * SP + shift[1][1]]);
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
// A warp computes PARAM_N output features x 32 lanes of four input features (neighbours, or 32 apart where rows are not aligned: two
// a lane were slower from eight rows on); a CTA stacks 8 warps along the output features. The prior variances are fetched
// before the rows are added up; the deltas come from shared memory, at one address for all lanes.
constexpr int PARAM_N = 8, PARAM_OUT = WARPS * PARAM_N;

// Four entries of a row, of which `left` follow from p on: neighbours (VEC: at least one is left), or 32 apart.
template <bool VEC>
__device__ __forceinline__ void load(const float *p, int left, float (&v)[4]) {
    if (VEC) {
        const float4 t = __ldg(reinterpret_cast<const float4 *>(p));
        v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
    } else {
#pragma unroll
        for (int c = 0; c < 4; c++) v[c] = c * 32 < left ? __ldg(p + c * 32) : 0.f;
    }
}

// weights pass by once: they are kept out of L1, where the rows are wanted
template <bool VEC>
__device__ __forceinline__ void load_once(const float *p, int left, float (&v)[4]) {
    if (VEC) {
        asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "l"(p));
    } else {
#pragma unroll
        for (int c = 0; c < 4; c++)
            if (c * 32 < left) asm volatile("ld.global.nc.L1::no_allocate.f32 %0, [%1];" : "=f"(v[c]) : "l"(p + c * 32));
    }
}

template <bool VEC>
__global__ void __launch_bounds__(THREADS, 2) grouped_few_param_kernel(const GroupedArgs a) {
    __shared__ __align__(16) float delta[FEW_PARAM_ROWS][2][PARAM_OUT];
    __shared__ int input[FEW_PARAM_ROWS];
    const int e = blockIdx.z;
    int r0, r1;
    expert_rows(a, e, r0, r1);
    const int rows = r1 - r0;
    if (rows > a.few) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, block_n = blockIdx.y * PARAM_OUT, n0 = block_n + warp * PARAM_N;
    constexpr int W = 4;
    const int k = blockIdx.x * 32 * W + (VEC ? lane * 4 : lane), left = a.K - k;
    float d[PARAM_N][W], v[PARAM_N][W], s[PARAM_N][W];
    const size_t o = ((size_t)e * a.N + n0) * a.K + k;
#pragma unroll
    for (int i = 0; i < PARAM_N; i++) {
#pragma unroll
        for (int c = 0; c < W; c++) d[i][c] = v[i][c] = s[i][c] = 0.f;
        if ((!VEC || left > 0) && rows > 0 && n0 + i < a.N) load_once<VEC>(a.var_w + o + (size_t)i * a.K, left, s[i]);
    }
    for (int i = threadIdx.x; i < rows * 2 * PARAM_OUT; i += THREADS) {
        const int n = block_n + i % PARAM_OUT, r = i / (2 * PARAM_OUT);
        const float *from = (i / PARAM_OUT) & 1 ? a.a1 : a.a0;
        delta[r][(i / PARAM_OUT) & 1][i % PARAM_OUT] = n < a.N ? __ldg(from + (size_t)(r0 + r) * a.N + n) : 0.f;
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
    if (left <= 0) return;
#pragma unroll 2
    for (int r = 0; r < rows; r++) {
        const int row = input[r];
        float x[W], q[W];
#pragma unroll
        for (int c = 0; c < W; c++) x[c] = 0.f;
        if (row >= 0) load<VEC>(a.x + (size_t)row * a.K + k, left, x);
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
        if (VEC) {
            __stcs(reinterpret_cast<float4 *>(p), make_float4(d[i][0], d[i][1], d[i][2], d[i][3]));
            __stcs(reinterpret_cast<float4 *>(u), make_float4(v[i][0], v[i][1], v[i][2], v[i][3]));
        } else {
#pragma unroll
            for (int c = 0; c < W; c++)
                if (c * 32 < left) p[c * 32] = d[i][c], u[c * 32] = v[i][c];
        }
    }
}

template <int PASS, bool VEC>
int launch_few(const GroupedArgs &a, cudaStream_t st) {
    constexpr size_t ring = stages(PASS) * (weights(PASS, VEC) + 2 * ROWS * SLAB), sums = WARPS * ROWS * 2 * OUT;
    constexpr size_t smem = (ring > sums ? ring : sums) * sizeof(float);
    // CTAs that have work, at most: as long as twice as many still run at the same time (two an SM), clusters cut the contraction,
    // into no less than 256 steps; the forward pass also beyond that, into no less than 2048. One row of one expert of 4096 x
    // 4096, forward, in 1 / 2 / 4 / 8 parts: 60 / 45 / 33 / 40 us; of two experts 78 / 56 / 56 / 69 us; of four 108 / 99 / 106 us.
    const int tiles = ((PASS == FWD ? a.N : a.K) + OUT - 1) / OUT, depth = PASS == FWD ? a.K : a.N;
    const long ctas = (long)tiles * (a.E < a.S ? a.E : a.S);
    int parts = 1;
    while (parts < 8 && depth >= 512 * parts && (ctas * parts <= 148 || (PASS == FWD && ctas * parts < 2 * 148 && depth >= 4096 * parts))) parts *= 2;
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
    const dim3 grid((a.K + 127) / 128, (a.N + PARAM_OUT - 1) / PARAM_OUT, a.E);
    if (vec) grouped_few_param_kernel<true><<<grid, THREADS, 0, st>>>(a);
    else grouped_few_param_kernel<false><<<grid, THREADS, 0, st>>>(a);
    TAGI_CUDA(cudaGetLastError());
    return TAGI_OK;
}

}  // namespace tagi
