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
// The mean and the variance are two accumulations over different operands (forward: mu_w.mu_a; mu_w^2.var_a followed by
// var_w.(mu_a^2 + var_a) as one contraction of twice the length), which neighbouring pairs do at the same time: mu_w is
// fetched from HBM for one and found in L2 by the other.
//
// Roles. Four warps fetch A from global memory into registers, four B (gathered rows, ragged edges and any alignment cost
// nothing extra there), a chunk at a time; they form squares, split, and store the parts to shared memory in the swizzled layouts
// the tensor core reads. Eight summing warps add each chunk's accumulator to their registers and write finished tiles out. One
// thread issues the MMAs, and a warp works out the items ahead of the others. Two slots of 64 contraction steps hold 2 x 96
// KiB of operands and two accumulators of 256 columns fill tensor memory; a slot's "full" barrier counts the converters
// (operands written) and the summing warps (accumulator read), its "done" barrier the MMAs' completion. Nothing stops at a
// tile's end: the next tile's operands are converted while the last one's chunks multiply and its sums are written.
//
// Bound by the tensor cores (and the power cap) from about 250 rows an expert on; by the converters with fewer (100 rows: 5000
// cycles a chunk, 1200 to issue its loads, 1500 until the values are there, 1200 to split and store them); by the output of
// the tiles in the parameter pass of few rows (12 bytes a weight).
#include "tagi_grouped_plan.cuh"
#include "tagi_grouped_split.cuh"

#include <cstddef>

namespace tagi {
namespace {

constexpr int SUMMERS = 8, CONVERTERS = 4, FIRST_B = SUMMERS + CONVERTERS, ISSUER = FIRST_B + CONVERTERS;   // warps (of A, and of B); then three more
constexpr int THREADS = 32 * (ISSUER + 4);
constexpr int WIDTH = 256, PER = WIDTH / 2;     // columns of a tile at most, and of a summing warp
constexpr int TASKS = 16;                       // times four values: a converter thread's part of its operand of a chunk
// Registers of a thread: all are launched with the same number; each warpgroup then takes what its role needs.
constexpr int LAUNCH_REGS = 96, SUMMER_REGS = 144, A_REGS = 80, B_REGS = 88, ISSUER_REGS = 24;
static_assert(SUMMERS * SUMMER_REGS + CONVERTERS * (A_REGS + B_REGS) + 4 * ISSUER_REGS <= (ISSUER + 4) * LAUNCH_REGS,
              "more registers than the launch has");
constexpr int KC = 64;                          // contraction steps of a chunk
constexpr uint32_t PART = 128 * KC * 2;         // one bf16 part of 128 rows (or columns) of a chunk: 16 KiB
constexpr uint32_t SLOT = 6 * PART;             // hi, mid, lo of A, then of B
constexpr uint32_t ACC = 256;                   // tensor-memory columns of a slot's accumulator
constexpr int PAIRS = 74;

__device__ int g_status;  // first wait that ran out, read and cleared by grouped_tc_status

struct Item {
    int chunks;                 // of the item; 0: there are no more items
    int e, m0, c0, cols, bn;    // expert; first feature; first column (output row, or feature in the parameter pass); live columns; width
    int kind, depth, p0, nk;    // MEAN or VAR; contraction length; first contraction row (parameter pass); chunks of one contraction
    int from, part;             // first chunk; WHOLE, or which of the pair's two partial sums the item goes to
};
// A warp of each CTA works out the items ahead of the others and hands them over through shared memory.
struct Record {
    Item item;
    int rows[128];              // forward pass: input rows of this CTA's columns, -1 where there is none
};
constexpr int RECORDS = 8;
constexpr int CUT_SAVES = 8;    // chunks that cutting has to save (see tagi_grouped_plan.cuh): it costs about 10 us, the time of four

struct Shared {                 // behind the slots
    uint64_t full[2], done[2], item_full[RECORDS], item_empty[RECORDS], turn;
    uint32_t tmem;
    volatile int abort_flag;
    Record record[RECORDS];
    alignas(16) int rows[4][16];      // parameter pass: input rows of a chunk's steps, per warp of A
    float aux[8][3][8][32];     // scale entries on their way to the summing warps: three groups of eight columns each
    float bias[128];            // parameter pass: sums of the deltas of this CTA's columns
    int start[2 * PAIRS + 2];   // of the tiles that are cut: chunks of those before each
    int before[];               // tiles of the experts before e, E + 1 entries
};
static_assert(offsetof(Shared, rows) % 16 == 0 && sizeof(Shared) % 8 == 0, "rows are read 16 bytes at a time");

// The mean or the variance of tile t.
template <int PASS>
__device__ __forceinline__ void tile_item(const GroupedArgs &a, const int *before, int t, int kind, Item &it) {
    it.kind = kind;
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
    const int n = l / mt, width = PASS == PARAM ? a.N : r1 - r0, nt = (width + WIDTH - 1) / WIDTH;
    it.bn = round_up((width + nt - 1) / nt, PASS == PARAM ? 128 : 32);
    it.cols = min(it.bn, width - n * it.bn);
    it.c0 = n * it.bn + (PASS == PARAM ? 0 : r0);
    it.p0 = r0;
    it.depth = PASS == FWD ? a.K : PASS == STATE ? a.N : r1 - r0;
    it.nk = (it.depth + KC - 1) / KC;
    it.chunks = PASS == FWD && kind == VAR ? 2 * it.nk : it.nk;
    it.from = 0;
    it.part = WHOLE;
}

// Item j of pair `pair`. Cut tiles: 3000 rows of 5 experts, 1001 to 1515 features, forward: 267 us whole, 216 us cut; 7288 rows of
// 2 experts, 16 to 75 features, parameter pass: 174 and 47 us.
template <int PASS>
__device__ __forceinline__ bool get_item(const GroupedArgs &a, Shared &sh, Plan &p, int pair, int pairs, int j, Item &it) {
    Share s;
    auto chunks_of = [&](int i) {
        Item t;
        tile_item<PASS>(a, sh.before, i >> 1, kind_of(i, pairs), t);
        return t.chunks;
    };
    if (!share_of(sh.start, p, pair, pairs, CUT_SAVES, j, chunks_of, s)) return false;
    tile_item<PASS>(a, sh.before, s.i >> 1, kind_of(s.i, pairs), it);
    if (s.chunks) it.from = s.from, it.chunks = s.chunks, it.part = s.part;
    return true;
}

// Operands of 128 rows x 64 contraction steps as the tensor core reads them (128-byte swizzle: 16-byte chunk c of line r
// lies at chunk c ^ (r & 7)), and which 16 groups of four values ("tasks") each of an operand's 128 threads brings there.
//  K-major: line = row, 64 steps of 2 bytes. Task t = 4 g + s: row g * 32 + row(), steps s * 16 + 0..3 + along(); a warp
//  loads 64 consecutive bytes of eight rows and stores to all banks.
//  MN-major: line = 64 rows of one step; the 64 lines of rows 0..63 come before those of rows 64..127. Task t: step
//  4 t + row(), rows along() + 0..3; a warp loads 512 consecutive bytes.
// Rows that are not aligned to 16 bytes are read a float at a time, and a warp's loads have to be neighbours all the same (the
// load unit takes a line of memory at a time). Neither the order of the steps nor that of the features matters to a sum:
//  forward pass, both operands: the order of step_at(); four lanes read neighbours.
//  state pass (WIDE), B: place 4 i + c of a line holds step i + 16 c, so that sixteen lanes read neighbours. Task t: row 8 t +
//  row(). A: its steps lie in the same order, and place 4 i + c of the CTA's 128 features holds feature i + 32 c. 3000 rows of 5
//  experts, 1001 to 1515 features: 168 us; 185 us without. In the other passes this was slower (forward: a thread then has
//  sixteen gathered rows; parameters: their output is scattered).
template <bool MN, bool SPREAD, bool WIDE>
struct Place {
    static constexpr uint32_t KSTEP = (MN ? 16 * 128 : 32) >> 4;             // 16 contraction steps, in 16-byte units
    static constexpr uint32_t LBO = MN ? 64 * 128 : 16;
    static constexpr bool LINE = !MN && WIDE;
    static constexpr int STRIDE = MN ? WIDE ? 32 : 1 : WIDE ? 16 : SPREAD ? 4 : 1;   // of a thread's four values along memory
    __device__ static int row(int warp, int lane) { return MN ? warp : LINE ? warp * 2 + (lane >> 4) : warp * 8 + ((lane >> 2) & 3) * 2 + (lane >> 4); }
    __device__ static int along(int lane) { return MN ? WIDE ? lane : lane * 4 : LINE ? lane & 15 : SPREAD ? lane & 3 : (lane & 3) * 4; }
    __device__ static uint32_t base(int warp, int lane) {
        const uint32_t r = row(warp, lane), c = (MN || LINE ? lane & 15 : lane & 3) >> 1;
        return (MN ? (lane >> 4) * 8192u : 0u) + r * 128 + ((c ^ (r & 7)) << 4) + (lane & 1) * 8;
    }
    // where task t goes, from base(): the swizzle's exclusive or with the bits of t that change the chunk or the line
    __device__ static uint32_t at(uint32_t base, int t) {
        return LINE ? base + t * 1024 : MN ? (base ^ ((t & 1) << 6)) + t * 512 : (base ^ ((t & 3) << 5)) + (t >> 2) * 4096;
    }
};
template <int PASS, bool VEC>
constexpr bool wide = !VEC && PASS == STATE;
template <int PASS, bool VEC>
using PlaceA = Place<PASS != FWD, !VEC && PASS == FWD, wide<PASS, VEC>>;
template <int PASS, bool VEC>
using PlaceB = Place<PASS == PARAM, !VEC && PASS == FWD, wide<PASS, VEC>>;
// Item j, as it was handed over; false when the CTA is aborting. release(): this warp needs the record no longer.
__device__ __forceinline__ bool take(Shared &sh, int j, Item &t) {
    t.chunks = 0;
    if (!mbar_wait(sh.item_full + j % RECORDS, (j / RECORDS) & 1, &sh.abort_flag, &g_status, ST_TIMEOUT_RAW)) return false;
    t = sh.record[j % RECORDS].item;
    return true;
}
__device__ __forceinline__ void release(Shared &sh, int j, int lane) {
    __syncwarp();
    if (lane == 0) mbar_arrive(sh.item_empty + j % RECORDS);
}

// What both operands' converters follow: the chunk that is loaded next. It runs ahead of the chunk that is stored.
struct Cursor {
    int j, c, end, kc;   // item; chunk, and the one behind the item's last (0: there are no more items); contraction step
    bool var, half;   // of a variance; second half of a forward variance (var_w . (mu_a^2 + var_a))
    __device__ void set(const Item &t, int item) {
        j = item, c = kc = end = 0, var = half = false;
        if (t.chunks == 0) return;   // the rest of such an item means nothing
        c = t.from, end = t.from + t.chunks;
        var = t.kind == VAR, half = t.from >= t.nk;   // only a forward variance has more than nk chunks
        kc = (half ? c - t.nk : c) * KC;
    }
};

using TcParts = Parts<256, 256>;

// A: 128 features of this CTA. A chunk is fetched whole as soon as the registers of the one before have been stored (one
// latency a chunk: loads that are waited for in turn would cost one each).
template <int PASS, bool VEC>
__device__ __forceinline__ void convert_a(const GroupedArgs &a, Shared &sh, int cta, int w, int lane, uint32_t smem_base) {
    constexpr bool MN = PASS != FWD, WIDE = wide<PASS, VEC>;
    using P = PlaceA<PASS, VEC>;
    const int row = P::row(w, lane), along = P::along(lane);
    const uint32_t to = smem_base + P::base(w, lane);
    float4 v[TASKS];
    Cursor cu;
    size_t base = 0;         // the thread's first element at contraction step 0, without the source
    int left = 0, nk = 0, depth = 0, p0 = 0;   // left: features from the thread's first one to the end (0: load nothing)
    int mine = -1;           // parameter pass: the input row that this lane looked up, of step 4 * lane + row of the cursor's chunk
    auto look_up = [&]() {
        if (PASS == PARAM) {
            const int k = cu.kc + (lane & 15) * 4 + row;
            mine = k < depth ? input_row(a, p0 + k) : -1;
        }
    };
    auto seek = [&](int j) {
        Item t;
        take(sh, j, t);
        release(sh, j, lane);
        cu.set(t, j);
        left = depth = 0;
        if (t.chunks == 0) return;
        const int m = t.m0 + cta * 128 + (MN ? along : row);
        base = PASS == FWD ? ((size_t)t.e * a.N + m) * a.K + along : PASS == STATE ? (size_t)t.e * a.N * a.K + m : m;
        left = (PASS == FWD ? a.N : a.K) - m;
        nk = t.nk, depth = t.depth, p0 = t.p0;
    };
    auto advance = [&]() {
        cu.kc += KC;
        if (++cu.c == cu.end) seek(cu.j + 1);
        else if (PASS == FWD && cu.c == nk) cu.kc = 0, cu.half = true;
        look_up();
    };
    auto load = [&]() {
        if (PASS == PARAM) {   // the looked up rows, for all lanes of the warp
            __syncwarp();
            if (lane < 16) sh.rows[w][lane] = mine;
            __syncwarp();
        }
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const float *src = PASS == FWD ? (cu.var && cu.half ? a.var_w : a.mu_w) + base + cu.kc + (size_t)(g * 32) * a.K
                               : PASS == STATE ? a.mu_w + base + (size_t)(cu.kc + (WIDE ? 0 : g * 16)) * a.K : a.x + base;
            int4 r = make_int4(-1, -1, -1, -1);
            if (PASS == PARAM) r = *reinterpret_cast<const int4 *>(&sh.rows[w][g * 4]);
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const int rs = s == 0 ? r.x : s == 1 ? r.y : s == 2 ? r.z : r.w;
                if (PASS == FWD) {
                    v[g * 4 + s] = ld4<VEC, P::STRIDE>(src + s * 16, g * 32 < left ? a.K - cu.kc - along - s * 16 : 0);
                } else if (PASS == STATE) {
                    const int k = WIDE ? row * 16 + g * 4 + s : s * 4 + row;   // place 16 g + 4 s + row; WIDE: step place / 4 + place % 4 * 16
                    v[g * 4 + s] = ld4<VEC, P::STRIDE>(src + (size_t)k * a.K, cu.kc + (WIDE ? 0 : g * 16) + k < a.N ? left : 0);
                } else {
                    v[g * 4 + s] = ld4<VEC>(src + (size_t)max(rs, 0) * a.K, rs >= 0 ? left : 0);
                }
            }
        }
    };
    seek(0);
    look_up();
    for (int i = 0; cu.end > 0; i++) {
        const int s = i & 1;
        const bool square = cu.var && !cu.half;
        load();
        advance();   // and looks up what the next load needs
        if (i >= 2 && !mbar_wait(sh.done + s, ((i - 2) >> 1) & 1, &sh.abort_flag, &g_status, ST_TIMEOUT_EMPTY)) return;
#pragma unroll
        for (int q = 0; q < TASKS; q++) store_split(P::at(to + s * SLOT, q), PART, square ? squared(v[q]) : v[q]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(sh.full + s, 0);
    }
}

// B: this CTA's half of the tile's columns, as A. In the parameter pass those are the deltas: the pairs of the first features'
// tile also add them up for the bias.
template <int PASS, bool VEC>
__device__ __forceinline__ void convert_b(const GroupedArgs &a, Shared &sh, int cta, int w, int lane, uint32_t smem_base) {
    constexpr bool MN = PASS == PARAM;
    using P = PlaceB<PASS, VEC>;
    const int row = P::row(w, lane), along = P::along(lane);
    const uint32_t to = smem_base + 3 * PART + P::base(w, lane);
    float4 v[TASKS];
    Cursor cu;
    int rows[4];             // forward pass: input rows of the thread's four columns
    size_t base = 0;         // state, parameter pass: the thread's first element at contraction step 0
    int left = 0, half_bn = 0, nk = 0, depth = 0;   // left: columns from the thread's first one to the end of the CTA's
    bool sum = false;        // the item's deltas are added up for the bias
    float4 total = make_float4(0.f, 0.f, 0.f, 0.f);
    uint32_t turn = 0;
    auto meet = [&]() {      // the four warps wait for one another
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.turn);
        return mbar_wait(&sh.turn, turn++ & 1, &sh.abort_flag, &g_status, ST_TIMEOUT_RAW);
    };
    auto seek = [&](int j) {
        Item t;
        take(sh, j, t);
        cu.set(t, j);
        half_bn = t.chunks ? t.bn >> 1 : 0;
        const int n = cta * half_bn + (MN ? along : row);
        left = t.chunks == 0 ? 0 : MN ? (along < half_bn ? t.cols - n : 0) : min(half_bn - row, t.cols - n);
        nk = t.nk, depth = t.chunks ? t.depth : 0;
        sum = PASS == PARAM && a.var_b != nullptr && t.chunks > 0 && t.m0 == 0;
        if (PASS == FWD) {
#pragma unroll
            for (int g = 0; g < 4; g++) rows[g] = g * 32 < left ? sh.record[j % RECORDS].rows[g * 32 + row] : -1;
        } else {
            base = PASS == STATE ? (size_t)(t.c0 + n) * a.N + along : (size_t)(t.p0 + row) * a.N + t.c0 + n;
        }
        if (PASS != PARAM) release(sh, j, lane);   // else when the item has ended
    };
    auto advance = [&]() {
        cu.kc += KC;
        if (++cu.c == cu.end) seek(cu.j + 1);
        else if (PASS == FWD && cu.c == nk) cu.kc = 0, cu.half = true;
    };
    auto load = [&](int g) {
        const float *src = PASS == FWD ? (!cu.var ? a.a0 : cu.half ? a.second : a.a1) + (size_t)max(rows[g], 0) * a.K + cu.kc + along
                                       : (cu.var ? a.a1 : a.a0) + base + (PASS == STATE ? (size_t)(g * 32) * a.N + cu.kc : (size_t)(cu.kc + g * 16) * a.N);
#pragma unroll
        for (int s = 0; s < 4; s++) {
            if (P::LINE) {
                v[g * 4 + s] = ld4<VEC, P::STRIDE>(src + (size_t)(s * 8) * a.N, g * 32 + s * 8 < left ? a.N - cu.kc - along : 0);
            } else if (PASS == FWD) {
                v[g * 4 + s] = ld4<VEC, P::STRIDE>(src + s * 16, rows[g] >= 0 ? a.K - cu.kc - along - s * 16 : 0);
            } else if (PASS == STATE) {
                v[g * 4 + s] = ld4<VEC>(src + s * 16, g * 32 < left ? a.N - cu.kc - along - s * 16 : 0);
            } else {
                v[g * 4 + s] = ld4<VEC>(src + (size_t)(s * 4) * a.N, cu.kc + (g * 4 + s) * 4 + row < depth ? left : 0);
            }
        }
    };
    seek(0);
    for (int i = 0; cu.end > 0; i++) {
        const int s = i & 1, lines = half_bn;
#pragma unroll
        for (int g = 0; g < 4; g++) load(g);
        const bool sums = PASS == PARAM && sum;
        const int ended = PASS == PARAM && cu.c + 1 == cu.end ? cu.j : -1;   // the item that ends with this chunk
        advance();
        if (i >= 2 && !mbar_wait(sh.done + s, ((i - 2) >> 1) & 1, &sh.abort_flag, &g_status, ST_TIMEOUT_EMPTY)) return;
#pragma unroll
        for (int g = 0; g < 4; g++)
            if (MN || g * 32 < lines) {   // narrow tiles have no columns for the later groups
#pragma unroll
                for (int q = g * 4; q < g * 4 + 4; q++)
                    if (MN ? along < round_up(lines, 64) : P::LINE ? q * 8 < lines : g * 32 + row < lines) store_split(P::at(to + s * SLOT, q), PART, v[q]);
            }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(sh.full + s, 0);
        if (PASS == PARAM && sums) {
#pragma unroll
            for (int q = 0; q < TASKS; q++) {
                add2(total.x, total.y, v[q].x, v[q].y);
                add2(total.z, total.w, v[q].z, v[q].w);
            }
        }
        if (ended >= 0) {
            if (sums) {
                const Item &t = sh.record[ended % RECORDS].item;
                float *b = sh.bias + along;
                for (int k = 0; k < 4; k++) {   // the four warps' sums, in the order of the warps
                    if (w == k) {
                        b[0] = total.x + (k ? b[0] : 0.f), b[1] = total.y + (k ? b[1] : 0.f);
                        b[2] = total.z + (k ? b[2] : 0.f), b[3] = total.w + (k ? b[3] : 0.f);
                    }
                    if (!meet()) return;
                }
                total = make_float4(0.f, 0.f, 0.f, 0.f);
                const int c = w * 32 + lane, n = cta * (t.bn >> 1) + c;
                if (c < t.bn >> 1 && t.part != WHOLE) {
                    TcParts::of(a, blockIdx.x >> 1, t.part)[TcParts::FLOATS + n] = sh.bias[c];
                } else if (c < t.bn >> 1 && n < t.cols) {
                    const size_t o = (size_t)t.e * a.N + t.c0 + n;
                    const float vb = __ldg(a.var_b + o);
                    (t.kind == VAR ? a.ob1 : a.ob0)[o] = t.kind == VAR ? vb * vb * sh.bias[c] : vb * sh.bias[c];
                }
                if (!meet()) return;   // read before the next item's sums are written
            }
            release(sh, ended, lane);
        }
    }
}

// Experts of more than `above` rows.
template <int PASS, bool VEC>
__global__ void __launch_bounds__(THREADS, 1) grouped_tc_kernel(const GroupedArgs a, int above) {
    constexpr bool A_MN = PASS != FWD, B_MN = PASS == PARAM;
    using PA = PlaceA<PASS, VEC>;   // layouts of the operands
    using PB = PlaceB<PASS, VEC>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    Shared &sh = *reinterpret_cast<Shared *>(smem_raw + (smem_base - smem_u32(smem_raw)) + 2 * SLOT);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cta = (int)cluster_ctarank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    if (warp == 0) {
        const int mt = ((PASS == FWD ? a.N : a.K) + 255) / 256;
        int carry = 0;
        for (int e0 = 0; e0 < a.E; e0 += 32) {
            int r0 = 0, r1 = 0;
            if (e0 + lane < a.E) expert_rows(a, e0 + lane, r0, r1);
            const int v = r1 - r0 > above ? mt * (((PASS == PARAM ? a.N : r1 - r0) + WIDTH - 1) / WIDTH) : 0;
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
    if (cta == 0 && threadIdx.x < 2) TcParts::piece(a, pairs, pair, threadIdx.x)->used = 0;
    if (sh.before[a.E] == 0) return;   // no expert of this size; the same in both CTAs
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; s++) {
            mbar_init(sh.full + s, 2 * ISSUER);   // counted in CTA 0
            mbar_init(sh.done + s, 1);                            // commit, multicast to both CTAs
        }
        for (int s = 0; s < RECORDS; s++) {
            mbar_init(sh.item_full + s, 1);
            mbar_init(sh.item_empty + s, ISSUER + (cta == 0));   // CTA 0: and the issuing thread
        }
        mbar_init(&sh.turn, 4);
        sh.abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == ISSUER) tmem_alloc_pair(&sh.tmem, 2 * ACC);
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();   // the peer's barriers exist before anyone arrives on them
    tc_fence_after_sync();
    const uint32_t tmem = sh.tmem;
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
            for (int j = 0; ok && take(sh, j, it) && it.chunks > 0; j++) {
                mbar_arrive(sh.item_empty + j % RECORDS);
                const uint32_t idesc = make_idesc_bf16(256, it.bn, A_MN, B_MN);
                for (int c = it.from; c < it.from + it.chunks; c++, i++) {
                    const int s = i & 1, left = it.depth - (c >= it.nk ? c - it.nk : c) * KC;
                    const int steps = wide<PASS, VEC> ? KC / 16 : max(1, min(KC / 16, (left + 15) / 16));
                    ok = mbar_wait_cluster(sh.full + s, (i >> 1) & 1, &sh.abort_flag, &g_status, ST_TIMEOUT_CONV);
                    if (!ok) break;
                    tc_fence_after_sync();
                    const uint32_t al = desc_lo(smem_base + s * SLOT, PA::LBO), bl = desc_lo(smem_base + s * SLOT + 3 * PART, PB::LBO);
                    const uint32_t d = tmem + s * ACC;
                    for (int k = 0; k < steps; k++) mma_small_products<(PART >> 4), (PART >> 4)>(d, al + k * PA::KSTEP, bl + k * PB::KSTEP, HI, idesc, k);
                    for (int k = 0; k < steps; k++) mma_large_product(d, al + k * PA::KSTEP, bl + k * PB::KSTEP, HI, idesc);
                    mma_commit_pair(sh.done + s);
                }
            }
        }
        if (warp == ISSUER + 1) {
            // ------------------------------------------------------------------------------------------------- items
            Plan plan = make_plan(PASS == FWD, 2 * sh.before[a.E], pairs, true);
            bool more = true;
            for (int j = 0; more; j++) {
                Record &r = sh.record[j % RECORDS];
                // the same for all lanes: they look at the rest together
                if (j >= RECORDS &&
                    !__all_sync(0xffffffffu, mbar_wait(sh.item_empty + j % RECORDS, (j / RECORDS - 1) & 1, &sh.abort_flag, &g_status, ST_TIMEOUT_EMPTY)))
                    break;
                Item t;
                more = get_item<PASS>(a, sh, plan, pair, pairs, j, t);
                if (!more) t.chunks = 0;
                if (more && t.part != WHOLE && cta == 0 && lane == 0)
                    *TcParts::piece(a, pairs, pair, t.part) = Piece{1, t.from + t.chunks == (PASS == FWD && t.kind == VAR ? 2 : 1) * t.nk, t.e, t.m0, t.c0, t.cols, t.bn, t.kind};
                if (lane == 0) r.item = t;
                if (PASS == FWD && more)
                    for (int l = lane; l < t.bn >> 1; l += 32) {
                        const int p = cta * (t.bn >> 1) + l;
                        r.rows[l] = p < t.cols ? input_row(a, t.c0 + p) : -1;
                    }
                __syncwarp();
                if (lane == 0) mbar_arrive(sh.item_full + j % RECORDS);
            }
        }
        __syncwarp();
        finish();
        if (warp == ISSUER) tmem_dealloc_pair(sh.tmem, 2 * ACC);
    } else if (warp < SUMMERS) {
        // ------------------------------------------------------------------------------------------- sums and output
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SUMMER_REGS));
        const int quad = warp & 3, group = warp >> 2;
        const uint32_t lane_addr = tmem + ((uint32_t)(quad * 32) << 16);
        float acc[PER];
#pragma unroll
        for (int x = 0; x < PER; x++) acc[x] = 0.f;
        if (lane == 0) {   // both accumulators are free
            mbar_arrive_cluster(sh.full, 0);
            mbar_arrive_cluster(sh.full + 1, 0);
        }
        const bool scaled = PASS == PARAM || (PASS == STATE && a.jcb != nullptr);
        const uint32_t aux_at = smem_u32(&sh.aux[warp][0][0][lane]);
        // Where a thread's part of a tile lies. Worked out from the record when it is needed (the record is kept until then):
        // the accumulators leave no registers to remember it in.
        struct Output {
            size_t base;   // first entry of the thread's column `first`
            int n, m, ld, kind, e;   // live columns of the warp's part; feature; pitch
            bool whole;
        };
        auto locate = [&](int j) {
            const volatile Item &t = sh.record[j % RECORDS].item;
            Output o;
            const int per = t.bn >> 1, first = group * per;
            o.n = min(per, t.cols - first);
            o.m = t.m0 + cta * 128 + feature_at(wide<PASS, VEC>, quad * 32 + lane);
            o.ld = PASS == FWD ? a.N : a.K;
            o.kind = t.kind, o.e = t.e;
            if (o.m >= o.ld) o.n = 0;
            o.whole = t.part == WHOLE;
            if (!o.whole) {   // a partial sum
                o.ld = 256;
                o.base = (size_t)(pair * 2 + t.part) * TcParts::PITCH + first * 256 + cta * 128 + quad * 32 + lane;
                return o;
            }
            o.base = ((PASS == PARAM ? (size_t)o.e * a.N : 0) + t.c0 + first) * o.ld + o.m;
            return o;
        };
        // Scale entries (Jacobian, prior variances) come from HBM and there are no registers to wait for them in either: a
        // lane copies its own to shared memory, 24 columns ahead, the first before the last chunk is done.
        auto fetch = [&](const Output &o, int g) {   // columns g .. g + 7
            if (scaled && o.whole) {
                const float *aux = (PASS == PARAM ? a.var_w : a.jcb) + o.base + (size_t)g * o.ld;
#pragma unroll
                for (int x = 0; x < 8; x++) copy_below(aux_at + ((g / 8 % 3) * 8 + x) * 128, aux + (size_t)x * o.ld, g + x, o.n);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        Item it;
        int i = 0;
        bool ok = true;
        for (int j = 0; ok && take(sh, j, it) && it.chunks > 0; j++) {
            const int per = it.bn >> 1, chunks = it.chunks;
            for (int c = 0; c < chunks; c++, i++) {
                const int s = i & 1;
                if (PASS != FWD && c == chunks - 1) {
                    const Output o = locate(j);
                    fetch(o, 0);
                    fetch(o, 8);
                    fetch(o, 16);
                }
                ok = mbar_wait(sh.done + s, (i >> 1) & 1, &sh.abort_flag, &g_status, ST_TIMEOUT_ACC);
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t at = lane_addr + s * ACC + group * per;
#pragma unroll
                for (int g = 0; g < PER; g += 8)
                    if (g < per) {
                        float v[8];
                        tmem_ld_32x8(at + g, v);
#pragma unroll
                        for (int x = 0; x < 8; x += 2) add2(acc[g + x], acc[g + x + 1], v[x], v[x + 1]);
                    }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(sh.full + s, 0);
            }
            if (!ok) break;
            const Output o = locate(j);
            release(sh, j, lane);
            float *out = (!o.whole ? a.parts : o.kind == VAR ? a.o1 : a.o0) + o.base;
            float bias = 0.f;
            if (PASS == FWD && a.mu_b && o.whole && o.n > 0) bias = __ldg((o.kind == VAR ? a.var_b : a.mu_b) + (size_t)o.e * a.N + o.m);
#pragma unroll
            for (int g = 0; g < PER; g += 8) {
                if (g >= o.n) break;
                if (PASS != FWD) asm volatile("cp.async.wait_group 2;" ::: "memory");
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    float z = acc[g + x];
                    if (PASS == FWD) z += bias;
                    float f = 1.f;
                    if (PASS != FWD && scaled) {   // a partial sum has none
                        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(aux_at + ((g / 8 % 3) * 8 + x) * 128));
                        f = o.whole ? f : 1.f;
                        z = o.kind == VAR ? z * f * f : z * f;
                    }
                    store_below(out + (size_t)x * o.ld, z, g + x, o.n);
                }
                out += (size_t)8 * o.ld;
                if (PASS != FWD) fetch(o, g + 24);
            }
            if (PASS != FWD) cp_async_wait_all();
#pragma unroll
            for (int x = 0; x < PER; x++) acc[x] = 0.f;
        }
        finish();
    } else {
        // ------------------------------------------------------------------------------------------------- converters
        if (warp < FIRST_B) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(A_REGS));
            convert_a<PASS, VEC>(a, sh, cta, warp - SUMMERS, lane, smem_base);
            finish();
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(B_REGS));
            convert_b<PASS, VEC>(a, sh, cta, warp - FIRST_B, lane, smem_base);
            finish();
        }
    }
}

// mu_a^2 + var_a, the forward variance's operand
__global__ void __launch_bounds__(256) grouped_second_moment_kernel(const float *__restrict__ mu, const float *__restrict__ var,
                                                                    size_t n, float *__restrict__ out) {
    const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i + 4 <= n) {
        const float4 m = __ldg(reinterpret_cast<const float4 *>(mu + i)), v = __ldg(reinterpret_cast<const float4 *>(var + i));
        *reinterpret_cast<float4 *>(out + i) =
            make_float4(fmaf(m.x, m.x, v.x), fmaf(m.y, m.y, v.y), fmaf(m.z, m.z, v.z), fmaf(m.w, m.w, v.w));
    } else {
        for (size_t j = i; j < n; j++) out[j] = fmaf(__ldg(mu + j), __ldg(mu + j), __ldg(var + j));
    }
}
__global__ void __launch_bounds__(256) grouped_second_moment_unaligned_kernel(const float *__restrict__ mu, const float *__restrict__ var,
                                                                              size_t n, float *__restrict__ out) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) out[i] = fmaf(__ldg(mu + i), __ldg(mu + i), __ldg(var + i));
}

template <int PASS>
int launch_pass(const GroupedArgs &a, int above, cudaStream_t st) {
    const bool vec = grouped_aligned(PASS, a);
    const size_t smem = 2 * SLOT + 1024 + sizeof(Shared) + (a.E + 1) * sizeof(int);
    const int pairs = grouped_tc_pairs(PASS, a.E, a.S, a.K, a.N);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * pairs);
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
    TAGI_CUDA(cudaLaunchKernelEx(&cfg, k, a, above));
    grouped_join_kernel<PASS, 256, 256><<<dim3(pairs, WIDTH / JOIN_COLUMNS), 256, 0, st>>>(a, pairs, vec ? wide<PASS, true> : wide<PASS, false>);
    TAGI_CUDA(cudaGetLastError());
    return TAGI_OK;
}
}  // namespace

// CTA pairs that may find work: one per SM pair, or as many as there can be chunks
int grouped_tc_pairs(int pass, int E, int S, int K, int N) {
    const int thin = pass == PARAM ? FEW_PARAM_ROWS : THIN_ROWS;
    const long mt = ((pass == FWD ? N : K) + 255) / 256, experts = E < S / (thin + 1) ? E : S / (thin + 1);   // at most as many have more rows
    const long tiles = mt * (pass == PARAM ? experts * ((N + 255) / 256) : S / 128 + experts);
    const long chunks = ((pass == FWD ? K : pass == STATE ? N : S) + KC - 1) / KC;
    const long most = tiles * chunks * (pass == FWD ? 3 : 2);
    return (int)(most < 1 ? 1 : most < PAIRS ? most : PAIRS);
}
size_t grouped_tc_parts_bytes(int pass, int E, int S, int K, int N) {
    return TcParts::bytes(grouped_tc_pairs(pass, E, S, K, N));
}

int grouped_second_moment(const GroupedArgs &a, cudaStream_t st) {
    const size_t n = (size_t)a.R * a.K;
    if (aligned16(a.a0) && aligned16(a.a1))
        grouped_second_moment_kernel<<<(unsigned)((n + 1023) / 1024), 256, 0, st>>>(a.a0, a.a1, n, a.second);
    else
        grouped_second_moment_unaligned_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a.a0, a.a1, n, a.second);
    TAGI_CUDA(cudaGetLastError());
    return TAGI_OK;
}

int grouped_tc(int pass, const GroupedArgs &a, cudaStream_t st) {
    if (pass == PARAM) return launch_pass<PARAM>(a, FEW_PARAM_ROWS, st);
    const int above = middle_likely(a.E, a.S) ? MIDDLE_ROWS : THIN_ROWS;   // what tagi_grouped_thin.cu has left
    if (a.S <= above) return TAGI_OK;
    return pass == FWD ? launch_pass<FWD>(a, above, st) : launch_pass<STATE>(a, above, st);
}

int grouped_tc_status(int *out, int reset) {
    TAGI_CUDA(cudaMemcpyFromSymbol(out, g_status, sizeof(int)));
    const int zero = 0;
    if (reset && *out) TAGI_CUDA(cudaMemcpyToSymbol(g_status, &zero, sizeof(int)));
    int thin = 0;
    const int rc = grouped_thin_status(&thin, reset);
    if (*out == 0) *out = thin;
    return rc;
}

}  // namespace tagi
