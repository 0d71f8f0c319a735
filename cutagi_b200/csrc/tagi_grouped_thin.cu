// Linear layers grouped by expert, forward and state pass of experts with 9 to 48 rows, and 49 to 128, on the tensor cores: the
// arithmetic of tagi_grouped_tc.cu for tiles so narrow that the weights' way from HBM and their conversion, not the
// multiplication, are what takes the time. Bound: HBM, 8 (forward) or 4 (state) bytes a weight.
//
// One CTA computes 128 features x all rows of an expert. The weights come through a ring of six to eight half-chunks (16 KiB
// each), so that about 100 KB of each SM are on their way from HBM whatever the converters do: by TMA, or with cp.async, by the
// 16-byte groups of memory that they lie in, where rows are not multiples of 16 bytes (30 rows of 4 experts of 2047 x 2047,
// forward: 100 us; of 2048 x 2048 66 us). Eight warps read them, a feature to a lane, and store the values' bf16 parts to tensor
// memory, where the MMAs take that operand from. Eight more fetch and split the rows, which come from L2; eight add up the
// accumulators of chunks of 64 steps; one issues the MMAs.
//
// Up to 48 rows the six products of 16 steps are three MMAs: the rows' parts lie below each other and count as one operand of up
// to 3 x 48 columns (STACKED). hi.[hi mid lo] adds to accumulators 0, 1 and 2, mid.[hi mid] to 1 and 2, lo.[hi] to 2: the
// accumulators hold the terms of one magnitude each and are added up when a chunk is read. The rows' warps take turns at the
// chunks (four for each: 365 us instead of 283 for 16 rows of 8 experts of 4096 x 4096, forward; HBM alone takes 164 us). With
// more rows the accumulators do not fit tensor memory three times, and the products are six MMAs into one.
#include "tagi_grouped_plan.cuh"
#include "tagi_grouped_split.cuh"
#include "tagi_tc_tile.cuh"

namespace tagi {
namespace {
namespace thin {

constexpr int SUMMERS = 8, CONVERT_A = 8, CONVERT_B = 8, LOADERS = 2;
constexpr int FIRST_A = SUMMERS, FIRST_B = FIRST_A + CONVERT_A, FIRST_LOADER = FIRST_B + CONVERT_B, ISSUER = FIRST_LOADER + LOADERS;
constexpr int THREADS = 32 * (ISSUER + 2);       // the last warp works out the items
constexpr int ROWS = 128, KC = 64, HALF = 32, MAX_RING = 8, RECORDS = 4, CTAS = 148;
// For tiles of up to COLS columns. STACKED: the rows' parts count as one operand.
template <int COLS>
struct Shape {
    static constexpr bool STACKED = COLS <= 48;
    static constexpr int ring(bool vec) { return STACKED ? 8 : vec ? 7 : 6; }   // half-chunks
    static constexpr uint32_t SLOT = 3 * COLS * KC * 2;   // the parts of a tile lie bn rows of 128 bytes apart
    // tensor-memory columns: two slots of accumulators, two slots of A's parts (two bf16 values a column)
    static constexpr uint32_t ACC = (STACKED ? 3 : 1) * COLS, A_COL = 2 * ACC;
    static_assert(SLOT % 1024 == 0, "the swizzle counts lines from multiples of 1024 bytes");
    static_assert(A_COL + 2 * 3 * (KC / 2) <= 512, "tensor memory");
};
// Registers of a thread, not stacked: all are launched with the same number; each warpgroup then takes what its role needs.
constexpr int LAUNCH_REGS = 72, SUMMER_REGS = 104, CONVERT_REGS = 64, OTHER_REGS = 40;
static_assert(SUMMERS * SUMMER_REGS + (CONVERT_A + CONVERT_B) * CONVERT_REGS + 4 * OTHER_REGS <= THREADS / 32 * LAUNCH_REGS, "more registers than the launch has");
// A half-chunk of weights. Lines that do not begin at multiples of 16 bytes take one 16-byte group more, begin up to three floats
// behind their place, and are not swizzled: a pitch of 36 floats keeps eight lines off each other's banks as well.
constexpr int FWD_PITCH = HALF + 4, STATE_PITCH = ROWS + 4;   // floats
__host__ __device__ constexpr uint32_t raw_bytes(bool vec) { return vec ? ROWS * HALF * 4 : ROWS * FWD_PITCH * 4; }
static_assert(HALF * STATE_PITCH * 4 <= raw_bytes(false), "");
constexpr uint32_t A_PART = KC / 2, A_SLOT = 3 * A_PART, TMEM_COLS = 512;
constexpr int CUT_SAVES = 12;   // chunks that cutting has to save (see tagi_grouped_plan.cuh): a chunk takes 1 us, cutting about 10

__device__ int g_status;  // first wait that ran out

struct Item {
    int chunks;                   // of the item; 0: there are no more items
    int e, m0, r0, rows, bn;      // expert; first feature; first row and their number; tile width
    int kind, depth, nk;          // MEAN or VAR; contraction length; chunks of one contraction
    int from, part;               // first chunk; WHOLE, or which of the CTA's two partial sums the item goes to
};
template <int COLS>
struct Shared {                   // behind the slots and the ring
    uint64_t full[2], done[2], raw_full[MAX_RING], raw_empty[MAX_RING], item_full[RECORDS], item_empty[RECORDS];
    uint32_t tmem;
    volatile int abort_flag;
    Item item[RECORDS];
    int input[RECORDS][COLS];     // forward: input rows of the item's columns, -1 where there is none
    int start[2 * CTAS + 2];      // of the tiles that are cut: chunks of those before each
    int before[];                 // tiles of the experts before e, E + 1 entries
};

// Item j of a CTA; chunks == 0: there is none.
template <int PASS, int COLS>
__device__ __forceinline__ void get_item(const GroupedArgs &a, Shared<COLS> &sh, Plan &p, int j, Item &it) {
    const int ctas = gridDim.x, *before = sh.before;
    it.depth = PASS == FWD ? a.K : a.N;
    it.nk = (it.depth + KC - 1) / KC;
    it.chunks = 0;
    Share s;
    auto chunks_of = [&](int i) { return PASS == FWD && kind_of(i, ctas) == VAR ? 2 * it.nk : it.nk; };
    if (!share_of(sh.start, p, blockIdx.x, ctas, CUT_SAVES, j, chunks_of, s)) return;
    const int t = s.i >> 1;
    it.kind = kind_of(s.i, ctas);
    int lo = 0, hi = a.E - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (before[mid] <= t) lo = mid; else hi = mid - 1;
    }
    it.e = lo;
    int r1;
    expert_rows(a, lo, it.r0, r1);
    it.rows = r1 - it.r0;
    it.m0 = (t - before[lo]) * ROWS;
    it.bn = round_up(it.rows, 16);
    it.from = s.from, it.part = s.part;
    it.chunks = s.chunks ? s.chunks : chunks_of(s.i);
}

template <int COLS>
__device__ __forceinline__ bool take(Shared<COLS> &sh, int j, Item &t) {
    t.chunks = 0;
    if (!mbar_wait(sh.item_full + j % RECORDS, (j / RECORDS) & 1, &sh.abort_flag, &g_status, ST_TIMEOUT_RAW)) return false;
    t = sh.item[j % RECORDS];
    return true;
}
template <int COLS>
__device__ __forceinline__ void release(Shared<COLS> &sh, int j, int lane) {
    __syncwarp();
    if (lane == 0) mbar_arrive(sh.item_empty + j % RECORDS);
}

__device__ __forceinline__ float4 lds4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

// 16 bytes to shared memory, the last 16 - `bytes` of them zero, if `on`: no branch.
__device__ __forceinline__ void copy16(uint32_t dst, const float *src, int bytes, bool on) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %3, 0;\n\t@p cp.async.cg.shared.global [%0], [%1], 16, %2;\n\t}" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"((int)on)
                 : "memory");
}
// of a 16-byte group before whose end lie `floats` of a line's floats (any number)
__device__ __forceinline__ int bytes_of(int floats) { return min(max(floats, 0), 4) * 4; }

// Experts of more than `above` and at most `upto` rows.
template <int PASS, bool VEC, int COLS>
__global__ void __launch_bounds__(THREADS, 1)
grouped_thin_kernel(const __grid_constant__ CUtensorMap mean_map, const __grid_constant__ CUtensorMap var_map, const GroupedArgs a, int above, int upto, bool may_cut) {
    using Sh = Shape<COLS>;
    using ThinParts = Parts<ROWS, COLS>;
    constexpr bool STACKED = Sh::STACKED;
    constexpr int RING = Sh::ring(VEC);
    constexpr uint32_t SLOT = Sh::SLOT, ACC = Sh::ACC, A_COL = Sh::A_COL;
    constexpr uint32_t RAW = raw_bytes(VEC);
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u, ring = smem_base + 2 * SLOT;
    Shared<COLS> &sh = *reinterpret_cast<Shared<COLS> *>(smem_raw + (smem_base - smem_u32(smem_raw)) + 2 * SLOT + RING * RAW);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 0) {
        const int mt = ((PASS == FWD ? a.N : a.K) + ROWS - 1) / ROWS;
        int carry = 0;
        for (int e0 = 0; e0 < a.E; e0 += 32) {
            int r0 = 0, r1 = 0;
            if (e0 + lane < a.E) expert_rows(a, e0 + lane, r0, r1);
            const int v = r1 - r0 > above && r1 - r0 <= upto ? mt : 0;
            int s = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += u;
            }
            if (e0 + lane < a.E) sh.before[e0 + lane] = carry + s - v;
            carry += __shfl_sync(0xffffffffu, s, 31);
        }
        if (lane == 0) sh.before[a.E] = carry;
    }
    __syncthreads();
    if (may_cut && threadIdx.x < 2) ThinParts::piece(a, gridDim.x, blockIdx.x, threadIdx.x)->used = 0;
    if (sh.before[a.E] == 0) return;   // no expert of this size
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; s++) {
            mbar_init(sh.full + s, SUMMERS + CONVERT_A + (STACKED ? CONVERT_B / 2 : CONVERT_B));   // stacked: B's take turns
            mbar_init(sh.done + s, 1);
        }
        for (int s = 0; s < RING; s++) {
            mbar_init(sh.raw_full + s, VEC ? 1 : LOADERS * 32);   // the thread that starts TMA, or every loading thread's copies
            mbar_init(sh.raw_empty + s, CONVERT_A / 2);   // and half of A's read a half-chunk
        }
        for (int s = 0; s < RECORDS; s++) {
            mbar_init(sh.item_full + s, 1);
            mbar_init(sh.item_empty + s, SUMMERS + CONVERT_A + CONVERT_B + LOADERS + 1);
        }
        sh.abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == ISSUER) tmem_alloc(&sh.tmem, TMEM_COLS);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = sh.tmem;

    if (warp < SUMMERS) {
        // -------------------------------------------------------------------------------------------- sums and output
        if (!STACKED) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SUMMER_REGS));
        const int quad = warp & 3, group = warp >> 2;
        const uint32_t lane_addr = tmem + ((uint32_t)(quad * 32) << 16);
        float acc[COLS / 2];
#pragma unroll
        for (int x = 0; x < COLS / 2; x++) acc[x] = 0.f;
        if (lane == 0) {   // both accumulators are free
            mbar_arrive(sh.full);
            mbar_arrive(sh.full + 1);
        }
        Item it;
        bool ok = true;
        for (int j = 0, i = 0; ok && take(sh, j, it) && it.chunks > 0; j++) {
            const int per = it.bn >> 1, first = group * per;   // multiples of 8
            for (int c = 0; c < it.chunks; c++, i++) {
                const int s = i & 1;
                ok = mbar_wait(sh.done + s, (i >> 1) & 1, &sh.abort_flag, &g_status, ST_TIMEOUT_ACC);
                if (!ok) break;
                tc_fence_after_sync();
#pragma unroll
                for (int g = 0; g < COLS / 2; g += 8)
                    if (g < per) {
                        float v[8], u[8], t[8];
                        if (!STACKED) {
                            tmem_ld_32x8(lane_addr + s * ACC + first + g, v);
#pragma unroll
                            for (int x = 0; x < 8; x += 2) add2(acc[g + x], acc[g + x + 1], v[x], v[x + 1]);
                            continue;
                        }
                        tmem_ld_32x8_async(lane_addr + s * ACC + 2 * it.bn + first + g, v);
                        tmem_ld_32x8_async(lane_addr + s * ACC + it.bn + first + g, u);
                        tmem_ld_32x8_async(lane_addr + s * ACC + first + g, t);
                        tmem_wait_ld(v, u, t);
#pragma unroll
                        for (int x = 0; x < 8; x += 2) {
                            add2(v[x], v[x + 1], u[x], u[x + 1]);
                            add2(v[x], v[x + 1], t[x], t[x + 1]);
                            add2(acc[g + x], acc[g + x + 1], v[x], v[x + 1]);
                        }
                    }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(sh.full + s);
            }
            if (!ok) break;
            const bool whole = it.part == WHOLE;
            const int m = it.m0 + quad * 32 + lane, features = PASS == FWD ? a.N : a.K, n = m < features ? min(per, it.rows - first) : 0,
                      ld = whole ? features : ROWS;
            const size_t base = (size_t)(it.r0 + first) * features + m;
            float *out = whole ? (it.kind == VAR ? a.o1 : a.o0) + base : ThinParts::of(a, blockIdx.x, it.part) + first * ROWS + quad * 32 + lane;
            float bias = 0.f;
            if (PASS == FWD && a.mu_b && whole && n > 0) bias = __ldg((it.kind == VAR ? a.var_b : a.mu_b) + (size_t)it.e * a.N + m);
            const bool scaled = PASS == STATE && a.jcb != nullptr && whole;
            float f[8];
#pragma unroll
            for (int x = 0; x < COLS / 2; x++) {
                if (x >= n) break;
                if (PASS == STATE && x % 8 == 0) {
#pragma unroll
                    for (int y = 0; y < 8; y++) f[y] = scaled && x + y < n ? __ldg(a.jcb + base + (size_t)(x + y) * ld) : 1.f;
                }
                float z = acc[x];
                if (PASS == FWD) z += bias;
                else z = it.kind == VAR ? z * f[x % 8] * f[x % 8] : z * f[x % 8];
                out[(size_t)x * ld] = z;
            }
#pragma unroll
            for (int x = 0; x < COLS / 2; x++) acc[x] = 0.f;
            release(sh, j, lane);
        }
    } else if (warp < FIRST_B) {
        // ------------------------------------------------------------------------------------------ weights, ring -> parts
        if (!STACKED) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CONVERT_REGS));
        // h: which half of each chunk
        const int w = warp - FIRST_A, quad = w & 3, h = w >> 2, row = quad * 32 + lane;
        Item it;
        bool ok = true;
        for (int j = 0, i = 0; ok && take(sh, j, it) && it.chunks > 0; j++) {
            release(sh, j, lane);
            int shift[4] = {};   // not aligned: of this lane's line (forward), of every fourth line (state)
            if (!VEC) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const size_t line = (size_t)it.e * a.N * a.K + (PASS == FWD ? (size_t)(it.m0 + row) * a.K : (size_t)k * a.K + it.m0);
                    shift[k] = PASS == FWD && k > 0 ? shift_of(a.var_w + line) : shift_of(a.mu_w + line);
                }
            }
            for (int c = it.from; c < it.from + it.chunks; c++, i++) {
                const int r = 2 * i + h, slot = i & 1;
                const uint32_t to = tmem + ((uint32_t)(quad * 32) << 16) + A_COL + slot * A_SLOT + h * (HALF / 2);
                const bool square = it.kind == VAR && (PASS == STATE || c < it.nk);
                // the slot first: once it is free, nothing that was to come before this half-chunk in its place of the ring is still to
                // come, so that the parity tells
                ok = (i < 2 || mbar_wait(sh.done + slot, ((i - 2) >> 1) & 1, &sh.abort_flag, &g_status, ST_TIMEOUT_EMPTY)) &&
                     mbar_wait(sh.raw_full + r % RING, (r / RING) & 1, &sh.abort_flag, &g_status, ST_TIMEOUT_RAW);
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t raw = ring + (r % RING) * RAW;
#pragma unroll
                for (int b = 0; b < HALF; b += 16) {   // sixteen steps at a time: two bf16 a column, eight columns a part
                    float v[16];
                    if (PASS == FWD && !VEC) {
                        const int s4 = c >= it.nk ? shift[1] : shift[0];
                        const bool one = s4 & 1, two = s4 & 2;
                        float u[20];
#pragma unroll
                        for (int q = 0; q < 5; q++) {
                            const float4 x = lds4(raw + row * (FWD_PITCH * 4) + (b + q * 4) * 4);
                            u[q * 4] = x.x, u[q * 4 + 1] = x.y, u[q * 4 + 2] = x.z, u[q * 4 + 3] = x.w;
                        }
#pragma unroll
                        for (int k = 0; k < 18; k++) u[k] = one ? u[k + 1] : u[k];
#pragma unroll
                        for (int k = 0; k < 16; k++) v[step_at<true>(k)] = two ? u[k + 2] : u[k];
                    } else if (PASS == FWD) {
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            const float4 x = lds4(raw + row * (HALF * 4) + (((b / 4 + q) ^ (row & 7)) << 4));
                            v[q * 4] = x.x, v[q * 4 + 1] = x.y, v[q * 4 + 2] = x.z, v[q * 4 + 3] = x.w;
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 16; k++)
                            asm volatile("ld.shared.f32 %0, [%1];"
                                         : "=f"(v[step_at<!VEC>(k)])   // its place (step_at is its own inverse)
                                         : "r"(raw + (b + k) * ((VEC ? ROWS : STATE_PITCH) * 4) + (row + shift[k & 3]) * 4)
                                         : "memory");
                    }
                    if (square) {
#pragma unroll
                        for (int k = 0; k < 16; k++) v[k] *= v[k];
                    }
#pragma unroll
                    for (int p = 0; p < 3; p++) {
                        float word[8];
#pragma unroll
                        for (int k = 0; k < 16; k += 2) {
                            word[k / 2] = __uint_as_float(top_halves(v[k], v[k + 1]));
                            if (p < 2) subtract_truncated2(v[k], v[k + 1]);
                        }
                        tmem_st_32x8(to + p * A_PART + b / 2, word);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(sh.raw_empty + r % RING);
                tmem_wait_st();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(sh.full + slot);
            }
        }
    } else if (warp < FIRST_LOADER) {
        // ------------------------------------------------------------------------------- rows, global memory -> parts
        // a warp loads 64 consecutive bytes of eight rows; two groups of four warps take turns at the chunks, or have half the rows
        if (!STACKED) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CONVERT_REGS));
        constexpr int TURNS = STACKED ? 2 : 1;
        const int w = (warp - FIRST_B) & 3, half = (warp - FIRST_B) >> 2, turn = STACKED ? half : 0;
        const int row = (STACKED ? 0 : half * 64) + w * 8 + ((lane >> 2) & 3) * 2 + (lane >> 4), along = VEC ? (lane & 3) * 4 : lane & 3;
        const uint32_t to = smem_base + row * 128 + ((((lane & 3) >> 1) ^ (row & 7)) << 4) + (lane & 1) * 8;
        float4 v[8];
        Item it;
        int in[2], j = 0, c = 0;   // c: the chunk that is loaded next
        bool ok = true;
        auto seek = [&]() {
            take(sh, j, it);
#pragma unroll
            for (int g = 0; g < 2; g++) {
                const int p = g * 32 + row;
                in[g] = it.chunks == 0 || p >= it.rows ? -1 : PASS == FWD ? sh.input[j % RECORDS][p] : it.r0 + p;
            }
            c = it.from;
            release(sh, j, lane);
        };
        auto load = [&]() {
            const bool second = PASS == FWD && c >= it.nk;
            const int kc = (second ? c - it.nk : c) * KC;
            const float *src = it.kind == MEAN ? a.a0 : second ? a.second : a.a1;
#pragma unroll
            for (int q = 0; q < 8; q++)
                v[q] = ld4<VEC, VEC ? 1 : 4>(src + (size_t)max(in[q >> 2], 0) * it.depth + kc + along + (q & 3) * 16,
                                in[q >> 2] >= 0 ? it.depth - kc - along - (q & 3) * 16 : 0);
        };
        auto step = [&]() {
            if (it.chunks > 0 && ++c == it.from + it.chunks) j++, seek();
        };
        seek();
        if (turn == 1) step();
        for (int i = turn; it.chunks > 0; i += TURNS) {
            const int s = i & 1, cols = it.bn;
            load();
            step();
            if (STACKED) step();
            if (i >= 2) ok = mbar_wait(sh.done + s, ((i - 2) >> 1) & 1, &sh.abort_flag, &g_status, ST_TIMEOUT_EMPTY);
            if (!ok) break;
#pragma unroll
            for (int q = 0; q < 8; q++)
                if ((q >> 2) * 32 + row < cols) store_split(((to + s * SLOT) ^ ((q & 3) << 5)) + (q >> 2) * 4096, cols * 128, v[q]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(sh.full + s);
        }
    } else if (!STACKED) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
    }
    // the warps that need few registers: a chain of its own, as all of a warpgroup's warps give registers back together
    if (warp < FIRST_LOADER) {
    } else if (warp < ISSUER) {
        // --------------------------------------------------------------------------------------- weights, HBM -> ring
        // Forward: lines of 32 steps of a feature, 16-byte chunk c of line l at c ^ (l & 7), which is what TMA's 128-byte
        // swizzle makes and what lets eight lanes read eight lines at once. State: lines of 128 features of a step.
        const int w = warp - FIRST_LOADER;
        Item it;
        bool ok = true;
        int r = 0;
        for (int j = 0; ok && take(sh, j, it) && it.chunks > 0; j++) {
            release(sh, j, lane);
            for (int c = it.from; ok && c < it.from + it.chunks; c++) {
                const bool second = PASS == FWD && c >= it.nk;
                const int kc = (second ? c - it.nk : c) * KC;
                for (int h = 0; h < 2; h++, r++) {
                    if (VEC && (w != 0 || lane != 0)) continue;
                    if (r >= RING) ok = mbar_wait(sh.raw_empty + r % RING, (r / RING - 1) & 1, &sh.abort_flag, &g_status, ST_TIMEOUT_EMPTY);
                    if (!ok) break;
                    const uint32_t dst = ring + (r % RING) * RAW;
                    const int k0 = kc + h * HALF;
                    if (VEC) {
                        mbar_arrive_expect_tx(sh.raw_full + r % RING, RAW);
                        tma_load_3d(dst, second ? &var_map : &mean_map, PASS == FWD ? k0 : it.m0, PASS == FWD ? it.m0 : k0, it.e, sh.raw_full + r % RING);
                        continue;
                    }
                    // 16-byte groups of lines: forward, 32 steps of a feature, by eight lanes; state, 128 features of a step, by a
                    // warp; then the lines' last groups. Lines eight (four) apart begin equally far from a multiple of 16 bytes.
                    const float *w0 = second ? a.var_w : a.mu_w, *safe = w0 - shift_of(w0);   // an address for copies of nothing
                    const float *src = w0 + (size_t)it.e * a.N * a.K + (size_t)(PASS == FWD ? it.m0 : k0) * a.K + (PASS == FWD ? k0 : it.m0);
                    const int lines = a.N - (PASS == FWD ? it.m0 : k0), live = a.K - (PASS == FWD ? k0 : it.m0), x = w * 32 + lane;
                    if (PASS == FWD) {
                        const int l = x >> 3, g = (x & 7) * 4;
                        const float *p = src + (size_t)l * a.K;
                        const int shift = shift_of(p), bytes = bytes_of(live + shift - g);
                        p += g - shift;
                        const uint32_t d = dst + (l * FWD_PITCH + g) * 4;
                        const bool begins = p < w0;   // the tensor begins within the group
                        if (begins)
                            for (int y = 1; y < 4; y++) cp_async_f32(d + y * 4, y >= shift ? p + y : w0, y >= shift && y < live + shift);
                        copy16(d, bytes ? p : safe, bytes, l < lines && !begins);
#pragma unroll
                        for (int i = 1; i < 16; i++) copy16(d + i * 8 * FWD_PITCH * 4, (bytes ? p : safe) + (bytes ? (size_t)i * 8 * a.K : 0), bytes, l + i * 8 < lines);
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const float *q = src + (size_t)(x + i * 64) * a.K;
                            const int n = bytes_of(live + shift_of(q) - HALF);
                            copy16(dst + ((x + i * 64) * FWD_PITCH + HALF) * 4, n ? q - shift_of(q) + HALF : safe, n, x + i * 64 < lines);
                        }
                    } else {
                        const int g = lane * 4;
                        const float *p = src + (size_t)w * a.K, *p2 = p + 2 * (size_t)a.K;
                        const int shift = shift_of(p), shift2 = shift_of(p2), bytes = bytes_of(live + shift - g), bytes2 = bytes_of(live + shift2 - g);
                        p += g - shift, p2 += g - shift2;
                        const uint32_t d = dst + (w * STATE_PITCH + g) * 4;
                        const bool begins = p < w0;
                        if (begins)
                            for (int y = 1; y < 4; y++) cp_async_f32(d + y * 4, y >= shift ? p + y : w0, y >= shift && y < live + shift);
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const int n = w + i * 2 < lines ? (i & 1 ? bytes2 : bytes) : 0;   // zeros for steps behind the last
                            copy16(d + i * 2 * STATE_PITCH * 4, n ? (i & 1 ? p2 : p) + (size_t)(i / 2 * 4) * a.K : safe, n, i > 0 || !begins);
                        }
                        if (w == 0) {
                            const float *q = src + (size_t)lane * a.K;
                            const int n = lane < lines ? bytes_of(live + shift_of(q) - ROWS) : 0;
                            copy16(dst + (lane * STATE_PITCH + ROWS) * 4, n ? q - shift_of(q) + ROWS : safe, n, true);
                        }
                    }
                    cp_async_arrive(sh.raw_full + r % RING);
                }
            }
        }
        // all copies have landed, unless the CTA gives up: then they are waited for here, again not for ever
        if (!VEC) cp_async_wait_all();
        else if (!ok || sh.abort_flag)
            for (int q = max(0, r - RING); w == 0 && lane == 0 && q < r; q++)
                for (int spin = 0; spin < 100000 && !mbar_try_wait(sh.raw_full + q % RING, (q / RING) & 1); spin++) {}
    } else if (warp == ISSUER) {
        // ------------------------------------------------------------------------------------------------------- MMA
        // the whole warp, with values that are the same in all lanes
        constexpr uint32_t HI = desc_hi(1024, SWZ_128B);
        const bool lead = elected();
        const uint32_t tm = uniform(tmem), base = uniform(smem_base);
        Item it;
        bool ok = true;
        // (also whether a wait has ended: lanes that part would wait for one another)
        for (int j = 0, i = 0; ok && __all_sync(0xffffffffu, take(sh, j, it) && it.chunks > 0); j++) {
            release(sh, j, lane);
            const int bn = uniform(it.bn), nk = uniform(it.nk), depth = uniform(it.depth), from = uniform(it.from), end = from + uniform(it.chunks);
            const uint32_t one = make_idesc_bf16(ROWS, bn, 0, 0), two = make_idesc_bf16(ROWS, 2 * bn, 0, 0), three = make_idesc_bf16(ROWS, 3 * bn, 0, 0);
            for (int c = from; c < end; c++, i++) {
                const int s = i & 1, left = depth - (c >= nk ? c - nk : c) * KC, steps = min(KC / 16, (left + 15) / 16);
                ok = __all_sync(0xffffffffu, mbar_wait(sh.full + s, (i >> 1) & 1, &sh.abort_flag, &g_status, ST_TIMEOUT_CONV));
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t x = tm + A_COL + s * A_SLOT, y = desc_lo(base + s * SLOT, 16), d = tm + s * ACC;
                if (STACKED) {
                    for (int k = 0; k < steps; k++)
                        mma_stacked_ts<A_PART>(d, d + bn, d + 2 * bn, x + k * 8, y + k * 2, HI, three, two, one, k, lead);
                } else {
                    for (int k = 0; k < steps; k++) mma_small_products_ts<A_PART>(d, x + k * 8, y + k * 2, bn * 8, HI, one, k, lead);
                    for (int k = 0; k < steps; k++) mma_large_product_ts(d, x + k * 8, y + k * 2, HI, one, lead);
                }
                if (lead) mma_commit(sh.done + s);
                __syncwarp();
            }
        }
    } else {
        // ----------------------------------------------------------------------------------------------------- items
        Plan plan = make_plan(PASS == FWD, 2 * sh.before[a.E], gridDim.x, may_cut);
        bool more = true;
        for (int j = 0; more; j++) {
            if (j >= RECORDS &&
                !__all_sync(0xffffffffu, mbar_wait(sh.item_empty + j % RECORDS, (j / RECORDS - 1) & 1, &sh.abort_flag, &g_status, ST_TIMEOUT_EMPTY)))
                break;
            Item t;
            get_item<PASS, COLS>(a, sh, plan, j, t);
            more = t.chunks > 0;
            if (more && t.part != WHOLE && lane == 0)
                *ThinParts::piece(a, gridDim.x, blockIdx.x, t.part) =
                    Piece{1, t.from + t.chunks == (PASS == FWD && t.kind == VAR ? 2 : 1) * t.nk, t.e, t.m0, t.r0, t.rows, t.bn, t.kind};
            if (lane == 0) sh.item[j % RECORDS] = t;
            if (PASS == FWD && more)
                for (int l = lane; l < t.rows; l += 32) sh.input[j % RECORDS][l] = input_row(a, t.r0 + l);
            __syncwarp();
            if (lane == 0) mbar_arrive(sh.item_full + j % RECORDS);
        }
    }
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == ISSUER) tmem_dealloc(tmem, TMEM_COLS);
}

// The weights [E][N][K] as boxes of one expert: 32 steps of 128 features (forward, swizzled) or 128 features of 32 steps
int make_map(int pass, const GroupedArgs &a, const float *w, CUtensorMap *map) {
    static EncodeTiledFn encode = tc_encode_fn();
    if (!encode) return fail(TAGI_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const cuuint64_t dims[3] = {(cuuint64_t)a.K, (cuuint64_t)a.N, (cuuint64_t)a.E}, strides[2] = {(cuuint64_t)a.K * 4, (cuuint64_t)a.K * a.N * 4};
    const cuuint32_t box[3] = {pass == FWD ? (cuuint32_t)HALF : (cuuint32_t)ROWS, pass == FWD ? (cuuint32_t)ROWS : (cuuint32_t)HALF, 1};
    const cuuint32_t step[3] = {1, 1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<float *>(w), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              pass == FWD ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? TAGI_OK : fail(TAGI_ERR_CUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
}

// CTAs, and whether tiles may be cut (which takes a second kernel, 5 us even if it finds nothing to do): where the items do not
// go once round the CTAs, if sharing them out saves 16 chunks; else if items are long and rounds few. 20 rows of one expert, 4096
// to 1000 features, forward: 122 us whole, 38 us cut.
struct Grid {
    int ctas;
    bool may_cut;
};
Grid grid_of(int pass, int above, int E, int S, int K, int N) {
    const long mt = ((pass == FWD ? N : K) + ROWS - 1) / ROWS, experts = E < S / (above + 1) ? E : S / (above + 1);
    const long items = 2 * mt * experts, nk = ((pass == FWD ? K : N) + KC - 1) / KC;   // experts with more than `above` rows, at most
    const long longest = pass == FWD ? 2 * nk : nk, chunks = pass == FWD ? items / 2 * 3 * nk : items * nk;
    const bool may_cut = items <= CTAS ? longest - chunks / CTAS >= 16 : items < 4 * CTAS && longest >= 48;
    const long most = may_cut ? chunks : items;
    return Grid{(int)(most < 1 ? 1 : most < CTAS ? most : CTAS), may_cut};
}

template <int PASS, int COLS>
int launch_thin(const GroupedArgs &a, int above, int upto, cudaStream_t st) {
    using Sh = Shape<COLS>;
    const bool vec = grouped_aligned(PASS, a);
    const size_t smem = 2 * Sh::SLOT + Sh::ring(vec) * raw_bytes(vec) + 1024 + sizeof(Shared<COLS>) + (a.E + 1) * sizeof(int);
    const Grid g = grid_of(PASS, above, a.E, a.S, a.K, a.N);
    CUtensorMap mean = {}, var = {};
    int rc;
    if (vec && (rc = make_map(PASS, a, a.mu_w, &mean)) != TAGI_OK) return rc;
    if (vec && PASS == FWD && (rc = make_map(PASS, a, a.var_w, &var)) != TAGI_OK) return rc;
    auto k = vec ? grouped_thin_kernel<PASS, true, COLS> : grouped_thin_kernel<PASS, false, COLS>;
    TAGI_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    k<<<g.ctas, THREADS, smem, st>>>(mean, var, a, above, upto, g.may_cut);
    TAGI_CUDA(cudaGetLastError());
    if (g.may_cut) {
        grouped_join_kernel<PASS, ROWS, COLS><<<dim3(g.ctas, COLS / JOIN_COLUMNS), ROWS, 0, st>>>(a, g.ctas, false);
        TAGI_CUDA(cudaGetLastError());
    }
    return TAGI_OK;
}

}  // namespace thin
}  // namespace

template <int PASS>
static int launch_all(const GroupedArgs &a, cudaStream_t st) {
    int rc = thin::launch_thin<PASS, 48>(a, a.few, THIN_ROWS, st);
    if (rc != TAGI_OK || !middle_likely(a.E, a.S)) return rc;
    return thin::launch_thin<PASS, 128>(a, THIN_ROWS, MIDDLE_ROWS, st);
}
int grouped_thin(int pass, const GroupedArgs &a, cudaStream_t st) { return pass == FWD ? launch_all<FWD>(a, st) : launch_all<STATE>(a, st); }

size_t grouped_thin_parts_bytes(int pass, int E, int S, int K, int N) {
    const thin::Grid g = thin::grid_of(pass, FEW_ROWS, E, S, K, N), h = thin::grid_of(pass, THIN_ROWS, E, S, K, N);
    const size_t x = g.may_cut ? Parts<thin::ROWS, 48>::bytes(g.ctas) : 0, y = middle_likely(E, S) && h.may_cut ? Parts<thin::ROWS, 128>::bytes(h.ctas) : 0;
    return x > y ? x : y;
}

int grouped_thin_status(int *out, int reset) {
    TAGI_CUDA(cudaMemcpyFromSymbol(out, thin::g_status, sizeof(int)));
    const int zero = 0;
    if (reset && *out) TAGI_CUDA(cudaMemcpyToSymbol(thin::g_status, &zero, sizeof(int)));
    return TAGI_OK;
}

}  // namespace tagi
