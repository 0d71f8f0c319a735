// Linear layers grouped by expert on the tcgen05 tensor cores, with the accuracy of 32-bit products.
//
// Arithmetic. A float is the exact sum of three bf16 numbers (8 + 8 + 8 bits of its significand: hi, mid, lo), so
// a * b = hi hi + (hi mid + mid hi) + mid mid + (hi lo + lo hi) up to 2^-24 |a b|: six bf16 products, each exact in the
// tensor core, on operands that keep the whole exponent range. The tensor core truncates each time it adds to its
// accumulator, so the contraction is cut into chunks of 64 that start from zero, the five small products of a chunk
// come before the large one, and chunks are added in registers with rounding: at most four truncations at full size in
// each. Measured error against 64 bits (2-norm, contractions of 1024 to 4096): 2.5e-7 on means and variances, where
// sums of 32-bit products give 3e-7 to 1.1e-6. Bound: the measured bf16 rate / 6 = 275 TFLOP/s.
//
// Shape of the work. Rows of the tensor-core tile are features (of the weights: always many), columns are the expert's
// rows (ragged: any width in steps of 32), so a thin expert costs a narrow tile. Two CTAs of a cluster share a tile of
// 256 features x up to 256 columns (cta_group::2); every accumulator lane is a feature, so stores run along memory.
// The mean and the variance are two accumulations over different operands (forward: mu_w.mu_a; var_w.(mu_a^2 + var_a)
// followed by mu_w^2.var_a as one contraction of twice the length), done one after the other by the same pair, which
// finds the second's operands in L2.
//
// Roles. Eight converter warps fetch both operands from global memory into registers (gathered rows, ragged edges and any
// alignment cost nothing extra there), form squares, split and store the parts to shared memory in the swizzled layouts
// the tensor core reads; half a chunk ahead is in flight. Eight summing warps add each chunk's accumulator to their
// registers and write finished tiles out. One thread issues the MMAs. Two slots of 64 contraction steps hold 2 x 96 KiB of
// operands and two accumulators of 256 columns fill tensor memory; a slot's "full" barrier counts the converters (operands
// written) and the summing warps (accumulator read), its "done" barrier the MMAs' completion. Nothing stops at a tile's
// end: the next tile's operands are converted while the last one's chunks multiply and its sums are written.
#include "tagi_grouped.h"
#include "tagi_tc_ptx.cuh"

namespace tagi {
namespace {

using namespace ptx;

constexpr int SUMMERS = 8, CONVERTERS = 8, ISSUER = SUMMERS + CONVERTERS;   // warps 0-7, 8-15, 16 (17-19 idle)
constexpr int THREADS = 32 * (ISSUER + 4);
// Registers of a thread: 640 threads are launched with 96 each; each warpgroup then takes what its role needs.
constexpr int LAUNCH_REGS = 96, SUMMER_REGS = 144, CONVERTER_REGS = 80, ISSUER_REGS = 24;
static_assert(SUMMERS * SUMMER_REGS + CONVERTERS * CONVERTER_REGS + 4 * ISSUER_REGS <= (ISSUER + 4) * LAUNCH_REGS,
              "more registers than the launch has");
constexpr int KC = 64;                          // contraction steps of a chunk
constexpr int TASKS = 8;                        // groups of four values a converter thread handles of each operand of a chunk
constexpr uint32_t PART = 128 * KC * 2;         // one bf16 part of 128 rows (or columns) of a chunk: 16 KiB
constexpr uint32_t SLOT = 6 * PART;             // hi, mid, lo of A, then of B
constexpr uint32_t ACC = 256;                   // tensor-memory columns of a slot's accumulator
constexpr int MEAN = 0, VAR = 1;
constexpr int PAIRS = 74;

__device__ int g_status;  // first wait that ran out, read and cleared by grouped_tc_status

struct Item {
    int e, m0, c0, cols, bn, kind, depth, p0, nk, chunks;
    // expert; first feature; first column (row of the output, or output feature in the parameter pass); live columns;
    // tile width; MEAN or VAR; contraction length; first contraction row (parameter pass); chunks of a contraction; of the item
};

__device__ __forceinline__ int round_up(int a, int b) { return (a + b - 1) / b * b; }

// Item j of pair `pair`. The two kinds of a tile are neighbours, so two pairs work on the same weights at the same time, and
// a pair's kinds alternate from one item to the next (in the forward pass a variance costs twice a mean).
template <int PASS>
__device__ __forceinline__ bool get_item(const GroupedArgs &a, const int *before, int pair, int pairs, int j, Item &it) {
    const int i = pair + j * pairs, t = i >> 1;
    if (t >= before[a.E]) return false;
    it.kind = (i + 2 * t / pairs) & 1;
    int lo = 0, hi = a.E - 1;   // the last expert whose tiles begin at or before t
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (before[mid] <= t) lo = mid; else hi = mid - 1;
    }
    it.e = lo;
    int r0, r1;
    expert_rows(a, lo, r0, r1);
    const int l = t - before[lo], mt = ((PASS == FWD ? a.N : a.K) + 255) / 256;
    it.m0 = (l % mt) * 256;
    const int n = l / mt, width = PASS == PARAM ? a.N : r1 - r0, nt = (width + 255) / 256;
    it.bn = round_up((width + nt - 1) / nt, PASS == PARAM ? 128 : 32);
    it.cols = min(it.bn, width - n * it.bn);
    it.c0 = n * it.bn + (PASS == PARAM ? 0 : r0);
    it.p0 = r0;
    it.depth = PASS == FWD ? a.K : PASS == STATE ? a.N : r1 - r0;
    it.nk = max(1, (it.depth + KC - 1) / KC);
    it.chunks = PASS == FWD && it.kind == VAR ? 2 * it.nk : it.nk;
    return true;
}

// Four consecutive floats, of which the first `valid` (0..4) exist. VEC: all four or none, 16-byte aligned.
template <bool VEC>
__device__ __forceinline__ float4 ld4(const float *p, int valid) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (VEC) {
        if (valid > 0) v = __ldg(reinterpret_cast<const float4 *>(p));
    } else {
        if (valid > 0) v.x = __ldg(p);
        if (valid > 1) v.y = __ldg(p + 1);
        if (valid > 2) v.z = __ldg(p + 2);
        if (valid > 3) v.w = __ldg(p + 3);
    }
    return v;
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
// hi, mid, lo of four values to their part tiles
__device__ __forceinline__ void store_split(uint32_t at, float4 v) {
    sts64(at, top_halves(v.x, v.y), top_halves(v.z, v.w));
    subtract_truncated2(v.x, v.y), subtract_truncated2(v.z, v.w);
    sts64(at + PART, top_halves(v.x, v.y), top_halves(v.z, v.w));
    subtract_truncated2(v.x, v.y), subtract_truncated2(v.z, v.w);
    sts64(at + 2 * PART, top_halves(v.x, v.y), top_halves(v.z, v.w));
}
__device__ __forceinline__ float4 squared(float4 v) { return make_float4(v.x * v.x, v.y * v.y, v.z * v.z, v.w * v.w); }

// kind::f16 instruction descriptor: FP32 accumulation, bf16 operands (see make_idesc_tf32 for the fields)
__host__ __device__ constexpr uint32_t make_idesc_bf16(int M, int N, int a_mn, int b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_bf16_pair(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                              uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "mov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %5, p;\n\t}"
        ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Operands of 128 rows x 64 contraction steps as the tensor core reads them (128-byte swizzle: 16-byte chunk c of line r
// lies at chunk c ^ (r & 7)).
//  K-major: line = row, 64 steps of 2 bytes. A lane loads 4 steps; 16 lanes fill a line.
//  MN-major: line = 64 rows of one step; the 64 lines of rows 0..63 come before those of rows 64..127.
template <bool MN>
struct Place {
    // line (row or step) and position (step or row) of the first of this thread's four tasks; tasks are LINES apart
    static constexpr int LINES = MN ? CONVERTERS : 2 * CONVERTERS;
    static constexpr uint32_t STRIDE = LINES * 128;
    static constexpr uint32_t KSTEP = (MN ? 16 * 128 : 32) >> 4;             // 16 contraction steps, in 16-byte units
    static constexpr uint32_t LBO = MN ? 64 * 128 : 16, SBO = 1024;
    // warp: 0 .. CONVERTERS - 1
    __device__ static int line(int warp, int lane) { return MN ? warp : warp * 2 + (lane >> 4); }
    __device__ static int along(int lane) { return MN ? lane * 4 : (lane & 15) * 4; }
    __device__ static uint32_t offset(int warp, int lane) {
        const uint32_t l = line(warp, lane), c = (lane & 15) >> 1;
        return (MN ? (lane >> 4) * 8192u : 0u) + l * 128 + ((c ^ (l & 7)) << 4) + (lane & 1) * 8;
    }
};

template <int PASS, bool VEC>
__global__ void __launch_bounds__(THREADS, 1) grouped_tc_kernel(const GroupedArgs a) {
    constexpr bool A_MN = PASS != FWD, B_MN = PASS == PARAM;
    using PA = Place<A_MN>;
    using PB = Place<B_MN>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *behind = smem_raw + (smem_base - smem_u32(smem_raw)) + 2 * SLOT;
    uint64_t *full = reinterpret_cast<uint64_t *>(behind), *done = full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + 2);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *before = reinterpret_cast<int *>(tmem_slot + 2);   // tiles of the experts before e, E + 1 entries

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cta = (int)cluster_ctarank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; s++) {
            mbar_init(full + s, 2 * (SUMMERS + CONVERTERS));   // counted in CTA 0
            mbar_init(done + s, 1);             // commit, multicast to both CTAs
        }
        *abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == ISSUER) tmem_alloc_pair(tmem_slot, 2 * ACC);
    if (warp == 0) {
        const int mt = ((PASS == FWD ? a.N : a.K) + 255) / 256;
        int carry = 0;
        for (int e0 = 0; e0 < a.E; e0 += 32) {
            int r0 = 0, r1 = 0;
            if (e0 + lane < a.E) expert_rows(a, e0 + lane, r0, r1);
            const int v = e0 + lane < a.E ? mt * (((PASS == PARAM ? a.N : r1 - r0) + 255) / 256) : 0;
            int s = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += u;
            }
            if (e0 + lane < a.E) before[e0 + lane] = carry + s - v;
            carry += __shfl_sync(0xffffffffu, s, 31);
        }
        if (lane == 0) before[a.E] = carry;
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();   // the peer's barriers exist before anyone arrives on them
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    // neither CTA frees tensor memory or leaves while the other may still signal or read it
    auto finish = [&]() {
        tc_fence_before_sync();
        __syncthreads();
        cluster_sync_all();
        tc_fence_after_sync();
    };

    if (warp >= ISSUER) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(ISSUER_REGS));
        // ---------------------------------------------------------------------------------------------- MMA (CTA 0)
        if (warp == ISSUER && lane == 0 && cta == 0) {
            constexpr uint32_t HI = desc_hi(1024, SWZ_128B);
            Item it;
            int i = 0;
            bool ok = true;
            for (int j = 0; ok && get_item<PASS>(a, before, pair, pairs, j, it); j++) {
                const uint32_t idesc = make_idesc_bf16(256, it.bn, A_MN, B_MN);
                for (int c = 0; c < it.chunks; c++, i++) {
                    const int s = i & 1, left = it.depth - (c >= it.nk ? c - it.nk : c) * KC;
                    const int steps = max(1, min(KC / 16, (left + 15) / 16));
                    ok = mbar_wait_cluster(full + s, (i >> 1) & 1, abort_flag, &g_status, ST_TIMEOUT_CONV);
                    if (!ok) break;
                    tc_fence_after_sync();
                    const uint32_t al = desc_lo(smem_base + s * SLOT, PA::LBO), bl = desc_lo(smem_base + s * SLOT + 3 * PART, PB::LBO);
                    const uint32_t d = tmem + s * ACC;
                    constexpr uint32_t P = PART >> 4;
                    uint32_t acc = 0;
                    for (int k = 0; k < steps; k++) {
                        const uint32_t x = al + k * PA::KSTEP, y = bl + k * PB::KSTEP;
                        mma_bf16_pair(d, x + 2 * P, HI, y, HI, idesc, acc);        // lo hi
                        acc = 1;
                        mma_bf16_pair(d, x, HI, y + 2 * P, HI, idesc, 1);          // hi lo
                        mma_bf16_pair(d, x + P, HI, y + P, HI, idesc, 1);          // mid mid
                        mma_bf16_pair(d, x + P, HI, y, HI, idesc, 1);              // mid hi
                        mma_bf16_pair(d, x, HI, y + P, HI, idesc, 1);              // hi mid
                    }
                    for (int k = 0; k < steps; k++) mma_bf16_pair(d, al + k * PA::KSTEP, HI, bl + k * PB::KSTEP, HI, idesc, 1);
                    mma_commit_pair(done + s);
                }
            }
        }
        __syncwarp();
        finish();
        if (warp == ISSUER) tmem_dealloc_pair(*tmem_slot, 2 * ACC);
    } else if (warp < SUMMERS) {
        // ------------------------------------------------------------------------------------------- sums and output
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SUMMER_REGS));
        const int quad = warp & 3, group = warp >> 2;
        const uint32_t lane_addr = tmem + ((uint32_t)(quad * 32) << 16);
        float acc[128];
#pragma unroll
        for (int x = 0; x < 128; x++) acc[x] = 0.f;
        if (lane == 0) {   // both accumulators are free
            mbar_arrive_cluster(full, 0);
            mbar_arrive_cluster(full + 1, 0);
        }
        Item it;
        int i = 0;
        bool ok = true;
        for (int j = 0; ok && get_item<PASS>(a, before, pair, pairs, j, it); j++) {
            const int per = it.bn >> 1;
            for (int c = 0; c < it.chunks; c++, i++) {
                const int s = i & 1;
                ok = mbar_wait(done + s, (i >> 1) & 1, abort_flag, &g_status, ST_TIMEOUT_ACC);
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t at = lane_addr + s * ACC + group * per;
#pragma unroll
                for (int g = 0; g < 128; g += 8)
                    if (g < per) {
                        float v[8];
                        tmem_ld_32x8(at + g, v);
#pragma unroll
                        for (int x = 0; x < 8; x += 2) add2(acc[g + x], acc[g + x + 1], v[x], v[x + 1]);
                    }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(full + s, 0);
            }
            if (!ok) break;
            const int m = it.m0 + cta * 128 + quad * 32 + lane, first = group * per, n = min(per, it.cols - first);
            const int ld = PASS == FWD ? a.N : a.K;
            const size_t base = ((PASS == PARAM ? (size_t)it.e * a.N : 0) + it.c0 + first) * ld + m;
            float *out = (it.kind == VAR ? a.o1 : a.o0) + base;
            const float *aux = PASS == PARAM ? a.var_w + base : PASS == STATE && a.jcb ? a.jcb + base : nullptr;
            const bool live = m < ld;
            float bias = 0.f;
            if (PASS == FWD && a.mu_b && live) bias = __ldg((it.kind == VAR ? a.var_b : a.mu_b) + (size_t)it.e * a.N + m);
#pragma unroll
            for (int g = 0; g < 128; g += 8) {
                if (g >= n || !live) break;
                float f[8];
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    f[x] = 1.f;
                    if (PASS != FWD && aux && g + x < n) f[x] = __ldg(aux + (size_t)(g + x) * ld);
                }
#pragma unroll
                for (int x = 0; x < 8; x++)
                    if (g + x < n) {
                        float z = acc[g + x];
                        if (PASS == FWD) z += bias;
                        else z = it.kind == VAR ? z * f[x] * f[x] : z * f[x];
                        out[(size_t)(g + x) * ld] = z;
                    }
            }
#pragma unroll
            for (int x = 0; x < 128; x++) acc[x] = 0.f;
        }
        finish();
    } else {
        // ------------------------------------------------------------------------------------------------- converters
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CONVERTER_REGS));
        const int w = warp - SUMMERS;
        const int a_line = PA::line(w, lane), a_along = PA::along(lane), b_line = PB::line(w, lane), b_along = PB::along(lane);
        const uint32_t a_off = smem_base + PA::offset(w, lane), b_off = smem_base + 3 * PART + PB::offset(w, lane);
        float4 va[TASKS], vb[4];
        // Loads run ahead of the conversion, into registers that were just stored: the item and chunk they belong to are
        // `nx` and `nc`. rows: the input rows that this lane looked up for its warp (gathered operands).
        Item nx;
        int nc = 0, nj = 0, a_rows = -1, b_rows = -1;
        bool more = get_item<PASS>(a, before, pair, pairs, 0, nx);

        auto chunk_k = [&](const Item &t, int c, int &half) {
            half = PASS == FWD && c >= t.nk;
            return (half ? c - t.nk : c) * KC;
        };
        auto look_up_a = [&]() {   // parameter pass: lane q < 8 knows the input row of step q * LINES + w of the chunk
            if (PASS == PARAM) {
                const int k = nc * KC + a_line + (lane & 7) * PA::LINES;
                a_rows = k < nx.depth ? input_row(a, nx.p0 + k) : -1;
            }
        };
        auto load_a = [&](int q0) {   // four tasks of the 128 features of this CTA
            int half;
            const int kc = chunk_k(nx, nc, half);
#pragma unroll
            for (int q = q0; q < q0 + 4; q++) {
                if (PASS == FWD) {
                    const int m = nx.m0 + cta * 128 + a_line + q * PA::LINES, k = kc + a_along;
                    const float *src = nx.kind == VAR && !half ? a.var_w : a.mu_w;
                    va[q] = ld4<VEC>(src + ((size_t)nx.e * a.N + m) * a.K + k, m < a.N ? a.K - k : 0);
                } else if (PASS == STATE) {
                    const int m = nx.m0 + cta * 128 + a_along, k = kc + a_line + q * PA::LINES;
                    va[q] = ld4<VEC>(a.mu_w + ((size_t)nx.e * a.N + k) * a.K + m, k < a.N ? a.K - m : 0);
                } else {
                    const int m = nx.m0 + cta * 128 + a_along, r = __shfl_sync(0xffffffffu, a_rows, q);
                    va[q] = ld4<VEC>(a.x + (size_t)max(r, 0) * a.K + m, r >= 0 ? a.K - m : 0);
                }
            }
        };
        auto look_up_b = [&]() {   // forward pass: lane knows the input row of column lane >> 1 of the warp's tasks
            if (PASS == FWD) {
                const int line = (lane >> 1) * PB::LINES + w * 2 + (lane & 1), half_bn = nx.bn >> 1, p = cta * half_bn + line;
                b_rows = lane < 2 * TASKS && line < half_bn && p < nx.cols ? input_row(a, nx.c0 + p) : -1;
            }
        };
        // one task of this CTA's half of the columns; second: the variances that belong to the means (forward pass)
        auto load_b = [&](int q, bool second) {
            int half;
            const int kc = chunk_k(nx, nc, half), half_bn = nx.bn >> 1, line = b_line + q * PB::LINES;
            if (PASS == PARAM) {
                const int k = kc + line, n = cta * half_bn + b_along;
                return ld4<VEC>((nx.kind == VAR ? a.a1 : a.a0) + (size_t)(nx.p0 + k) * a.N + nx.c0 + n,
                                k < nx.depth && b_along < half_bn ? nx.cols - n : 0);
            }
            const int k = kc + b_along;
            if (PASS == FWD) {
                const int r = __shfl_sync(0xffffffffu, b_rows, q * 2 + (lane >> 4));
                return ld4<VEC>((second || (nx.kind == VAR && half) ? a.a1 : a.a0) + (size_t)max(r, 0) * a.K + k, r >= 0 ? a.K - k : 0);
            }
            const int p = cta * half_bn + line;
            return ld4<VEC>((nx.kind == VAR ? a.a1 : a.a0) + (size_t)(nx.c0 + p) * a.N + k, line < half_bn && p < nx.cols ? a.N - k : 0);
        };
        // vb: four tasks from q0, or (sums) the means and variances of two
        auto load_b4 = [&](int q0, bool sums) {
            if (PASS == FWD && sums) {
                vb[0] = load_b(q0, false), vb[1] = load_b(q0 + 1, false);
                vb[2] = load_b(q0, true), vb[3] = load_b(q0 + 1, true);
            } else {
#pragma unroll
                for (int q = 0; q < 4; q++) vb[q] = load_b(q0 + q, false);
            }
        };
        bool ok = true;
        if (more) {
            look_up_a();
            look_up_b();
            load_b4(0, PASS == FWD && nx.kind == VAR);
            load_a(0);
            load_a(4);
        }
        for (int i = 0; ok && more; i++) {
            const int s = i & 1;
            int half;
            chunk_k(nx, nc, half);
            const bool sums = PASS == FWD && nx.kind == VAR && !half, square = nx.kind == VAR && !sums;
            const int lines = PASS == PARAM ? round_up(nx.bn >> 1, 64) : nx.bn >> 1;   // columns that this CTA holds
            if (i >= 2) {
                ok = mbar_wait(done + s, ((i - 2) >> 1) & 1, abort_flag, &g_status, ST_TIMEOUT_EMPTY);
                if (!ok) break;
            }
            auto store_a = [&](int q0) {
#pragma unroll
                for (int q = q0; q < q0 + 4; q++)
                    store_split(a_off + s * SLOT + q * PA::STRIDE, square ? squared(va[q]) : va[q]);
            };
            auto store_b = [&](int q, float4 v) {
                if (PASS == PARAM ? b_along < lines : b_line + q * PB::LINES < lines) store_split(b_off + s * SLOT + q * PB::STRIDE, v);
            };
            auto store_b4 = [&](int q0) {
                if (PASS == FWD && sums) {
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        const float4 x = vb[q], v = vb[q + 2];
                        store_b(q0 + q, make_float4(fmaf(x.x, x.x, v.x), fmaf(x.y, x.y, v.y), fmaf(x.z, x.z, v.z), fmaf(x.w, x.w, v.w)));
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < 4; q++) store_b(q0 + q, vb[q]);
                }
            };
            // Every load is issued two groups of stores before its values are needed. With sums, columns take twice the
            // registers: they come in four groups, the last two of this chunk (the next cannot be looked up earlier).
            store_b4(0);
            load_b4(sums ? 2 : 4, sums);
            if (PASS == FWD && sums) {
                store_a(0);
                store_b4(2);
                load_b4(4, true);
                store_a(4);
                store_b4(4);
                load_b4(6, true);
            } else {
                store_a(0);
                store_a(4);
            }
            Item cur_next = nx;   // the next chunk's item
            int c_next = nc + 1, j_next = nj;
            bool has_next = true;
            if (c_next == nx.chunks) {
                c_next = 0;
                has_next = get_item<PASS>(a, before, pair, pairs, ++j_next, cur_next);
            }
            store_b4(sums ? 6 : 4);
            nx = cur_next, nc = c_next, more = has_next;
            if (more) {
                look_up_a();
                if (j_next != nj) look_up_b();
                load_b4(0, PASS == FWD && nx.kind == VAR && nc < nx.nk);
                load_a(0);
                load_a(4);
            }
            nj = j_next;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(full + s, 0);
        }
        finish();
    }
}

template <int PASS>
int launch_pass(const GroupedArgs &a, cudaStream_t st) {
    const bool vec = a.K % 4 == 0 && a.N % 4 == 0 && aligned16(a.mu_w) && aligned16(a.var_w) && aligned16(a.a0) && aligned16(a.a1) &&
                     aligned16(a.x);
    const size_t smem = 2 * SLOT + 1024 + 64 + (a.E + 1) * sizeof(int);
    const long mt = ((PASS == FWD ? a.N : a.K) + 255) / 256;
    const long most = 2 * mt * (PASS == PARAM ? (long)a.E * ((a.N + 255) / 256) : a.S / 256 + (a.E < a.S ? a.E : a.S));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (unsigned)(most < PAIRS ? most : PAIRS));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    auto k = vec ? grouped_tc_kernel<PASS, true> : grouped_tc_kernel<PASS, false>;
    TAGI_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    TAGI_CUDA(cudaLaunchKernelEx(&cfg, k, a));
    return TAGI_OK;
}

}  // namespace

int grouped_tc(int pass, const GroupedArgs &a, cudaStream_t st) {
    return pass == FWD ? launch_pass<FWD>(a, st) : pass == STATE ? launch_pass<STATE>(a, st) : launch_pass<PARAM>(a, st);
}

int grouped_tc_status(int *out, int reset) {
    TAGI_CUDA(cudaMemcpyFromSymbol(out, g_status, sizeof(int)));
    const int zero = 0;
    if (reset && *out) TAGI_CUDA(cudaMemcpyToSymbol(g_status, &zero, sizeof(int)));
    return TAGI_OK;
}

}  // namespace tagi
