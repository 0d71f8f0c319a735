// Routing of tokens to experts: the k best experts of every token by the means of the router's scores, the moments of the
// softmax over the chosen scores (the gates), and the dispatch order, a stable counting sort of the token's slots by expert.
// The backward pass takes deltas of the gates to deltas of the scores.
//
// A group of 8, 16 or 32 lanes ranks one token, so a warp up to four: the kernel is bound by the instructions it issues
// (32768 tokens, 128 experts, 8 chosen: a token per warp took 574 of them and 28 us; four per warp 306 and 17 us). Each lane
// keeps E / G neighbouring experts' scores as order-preserving integers in sorted groups of four; a round takes the largest
// head over the group's lanes, the lowest lane and four that hold it (ties go to the lowest index), and moves that four up.
// The counting sort cuts the tokens into blocks. The first kernel also counts its block's slots per expert; the second
// adds up the counts of the blocks before its own and ranks its slots with warp matches. Nothing depends on the order in
// which warps run: shared-memory atomics only add integers. Up to ONE_BLOCK_TOKENS tokens both halves are one launch of
// one block.
#include "tagi_common.h"

#include <type_traits>

namespace tagi {
namespace {

constexpr int MAX_EXPERTS = 1024, MAX_K = 32, MAX_TOKENS = 1 << 30;
// Warps of a block: the more the shorter the chain of tokens that a warp ranks one after the other (a block per SM holds
// them all), as far as the per-warp counts fit shared memory and a lane's scores its registers.
__host__ __device__ constexpr int warps_for(int E) { return E <= 256 ? 32 : 8; }
constexpr int ONE_BLOCK_TOKENS = 32;
constexpr int MAX_BLOCKS = 148;
constexpr unsigned FULL = 0xffffffffu;

struct RouteArgs {
    int T, E, k, per_block;  // tokens of a block
    const float *mu_s, *var_s;
    int *expert;
    float *mu_g, *var_g;
    int *offsets, *token, *pos;
    int *counts;  // [blocks][E]
    bool vec;     // rows of scores are aligned to 16 bytes
};

// Order-preserving integer of a score; 0 for the scores that bar an expert (-inf, NaN). -0 counts as 0.
__device__ __forceinline__ unsigned score_key(float s) {
    if (!(s > -INFINITY)) return 0u;
    const unsigned u = __float_as_uint(s + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_score(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

// Ranks the tokens [t0, t1) of the block, G lanes to a token, writes their slots' experts and gates and adds the slots to
// count[e]. Lane l of a group holds experts l * EPL .. l * EPL + EPL - 1.
template <int G, int EPL, int WARPS>
__device__ __forceinline__ void rank_tokens(const RouteArgs &a, long t0, long t1, int *count) {
    constexpr int FOURS = EPL / 4, TOKENS = 32 / G;
    const int lane = threadIdx.x & 31, l = lane & (G - 1), first = l * EPL, shift = lane & ~(G - 1);
    const bool vec = a.vec;
    for (long step = t0 + (threadIdx.x >> 5) * TOKENS; step < t1; step += WARPS * TOKENS) {
        const long t = step + lane / G;
        const bool live = t < t1;
        const float *score = a.mu_s + t * a.E + first;
        unsigned key[FOURS][4], order[FOURS];   // order: places of the four within it, a byte each
#pragma unroll
        for (int c = 0; c < FOURS; c++) {
            float f[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (vec) {
                if (live && first + c * 4 < a.E) {
                    const float4 x = __ldg(reinterpret_cast<const float4 *>(score) + c);
                    f[0] = x.x, f[1] = x.y, f[2] = x.z, f[3] = x.w;
                }
            } else {
#pragma unroll
                for (int q = 0; q < 4; q++)
                    if (live && first + c * 4 + q < a.E) f[q] = __ldg(score + c * 4 + q);
            }
#pragma unroll
            for (int q = 0; q < 4; q++) key[c][q] = score_key(f[q]);
        }
#pragma unroll
        for (int c = 0; c < FOURS; c++) {   // only neighbours are exchanged, and only if out of order: equal keys keep theirs
            unsigned at[4] = {0u, 1u, 2u, 3u};
#pragma unroll
            for (int end = 3; end > 0; end--)
#pragma unroll
                for (int q = 0; q < end; q++) {
                    const unsigned x = key[c][q], y = key[c][q + 1], i = at[q], j = at[q + 1];
                    const bool swap = y > x;
                    key[c][q] = max(x, y), key[c][q + 1] = min(x, y);
                    at[q] = swap ? j : i, at[q + 1] = swap ? i : j;
                }
            order[c] = at[0] | at[1] << 8 | at[2] << 16 | at[3] << 24;
        }
        int mine = -1;   // slot l: its expert and score
        unsigned chosen = 0u;
        for (int j = 0; j < a.k; j++) {
            unsigned head = key[0][0];
#pragma unroll
            for (int c = 1; c < FOURS; c++) head = max(head, key[c][0]);
            unsigned best = head;
            if (G == 32) {
                best = __reduce_max_sync(FULL, head);
            } else {
#pragma unroll
                for (int o = G / 2; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(FULL, best, o));
            }
            const unsigned holders = __ballot_sync(FULL, head == best) >> shift;   // the group's lowest lane is the lowest bit
            const int winner = __ffs(holders) - 1;
            bool take = l == winner;
            unsigned at = 0u;
#pragma unroll
            for (int c = 0; c < FOURS; c++) {
                if (take && key[c][0] == best) {
                    at = c * 4 + (order[c] & 255u);
                    key[c][0] = key[c][1], key[c][1] = key[c][2], key[c][2] = key[c][3], key[c][3] = 0u;
                    order[c] >>= 8;
                    take = false;
                }
            }
            at = __shfl_sync(FULL, at + first, winner, G);
            if (l == j && best != 0u) mine = (int)at, chosen = best;   // 0: the experts left are barred
        }
        const float s = mine < 0 ? -INFINITY : key_score(chosen);
        // softmax over the chosen scores (slot 0 holds the largest); equal infinite scores share evenly
        const float top = __shfl_sync(FULL, s, 0, G);
        const float p = mine < 0 ? 0.f : s == top ? 1.f : expf(s - top);
        float z = p;
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) z += __shfl_xor_sync(FULL, z, o);
        const float g = mine < 0 ? 0.f : p / z;
        const float v = mine < 0 || a.var_s == nullptr ? 0.f : __ldg(a.var_s + t * a.E + mine);
        // var_g_i = g_i^2 ((1 - g_i)^2 v_i + sum_{j != i} g_j^2 v_j); 1 - g_i as the sum of the others does not cancel
        float rest = 0.f, others = 0.f;
        for (int j = 0; j < a.k; j++) {
            const float gj = __shfl_sync(FULL, g, j, G), vj = __shfl_sync(FULL, v, j, G);
            if (j != l) rest += gj, others += gj * gj * vj;
        }
        if (live && l < a.k) {
            const long i = t * a.k + l;
            a.expert[i] = mine;
            a.mu_g[i] = g;
            a.var_g[i] = g * g * (rest * rest * v + others);
            if (mine >= 0) atomicAdd(count + mine, 1);
        }
    }
}

// Exclusive sum over the experts of total[e], in place; total[E] receives the sum. Called by the whole block.
__device__ __forceinline__ void exclusive_sum(int *total, int E) {
    if (threadIdx.x < 32) {
        int carry = 0;
        for (int e0 = 0; e0 < E; e0 += 32) {
            const int e = e0 + threadIdx.x, v = e < E ? total[e] : 0;
            int s = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(FULL, s, o);
                if ((int)threadIdx.x >= o) s += u;
            }
            if (e < E) total[e] = carry + s - v;
            carry += __shfl_sync(FULL, s, 31);
        }
        if (threadIdx.x == 0) total[E] = carry;
    }
    __syncthreads();
}

// Positions of the slots [i0, i1) of this block. base[e] is where the block's first slot of expert e goes. Each warp
// takes a contiguous segment: it counts, the counts of the warps before it are added, then it ranks 32 slots at a time.
template <int WARPS>
__device__ __forceinline__ void place_slots(const RouteArgs &a, long i0, long i1, const int *base, int *warp_count) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int *mine = warp_count + warp * a.E;
    for (int e = threadIdx.x; e < WARPS * a.E; e += WARPS * 32) warp_count[e] = 0;
    __syncthreads();
    const long seg = ((i1 - i0 + WARPS - 1) / WARPS + 31) / 32 * 32, s0 = min(i1, i0 + warp * seg), s1 = min(i1, s0 + seg);
    for (long i = s0 + lane; i < s1; i += 32) {
        const int e = a.expert[i];
        if (e >= 0) atomicAdd(mine + e, 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += WARPS * 32) {
        int s = base[e];
        for (int w = 0; w < WARPS; w++) {
            const int c = warp_count[w * a.E + e];
            warp_count[w * a.E + e] = s;
            s += c;
        }
    }
    __syncthreads();
    for (long i = s0; i < s1; i += 32) {   // the segment is a whole number of 32s except at its end: all lanes stay in step
        const int e = i + lane < s1 ? a.expert[i + lane] : -1;
        const unsigned same = __match_any_sync(FULL, e);
        int p = -1;
        if (e >= 0) p = mine[e] + __popc(same & ((1u << lane) - 1u));
        __syncwarp();
        if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
        __syncwarp();
        if (i + lane < s1) {
            a.pos[i + lane] = p;
            if (p >= 0) a.token[p] = (int)((unsigned)(i + lane) / (unsigned)a.k);
        }
    }
}

// slots without an expert leave the end of `token` empty
__device__ __forceinline__ void clear_tail(const RouteArgs &a, long live, long first, long stride) {
    for (long i = live + first; i < (long)a.T * a.k; i += stride) a.token[i] = -1;
}

template <int G, int EPL, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) route_rank_kernel(const RouteArgs a) {
    extern __shared__ int count[];
    const long t0 = (long)blockIdx.x * a.per_block, t1 = min((long)a.T, t0 + a.per_block);
    for (int e = threadIdx.x; e < a.E; e += WARPS * 32) count[e] = 0;
    __syncthreads();
    rank_tokens<G, EPL, WARPS>(a, t0, t1, count);
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += WARPS * 32) a.counts[(long)blockIdx.x * a.E + e] = count[e];
}

template <int WARPS>
__global__ void __launch_bounds__(WARPS * 32) route_place_kernel(const RouteArgs a) {
    extern __shared__ int sh[];  // total [E + 1], before [E], warp counts [WARPS][E]
    int *total = sh, *before = sh + a.E + 1, *warp_count = before + a.E;
    for (int e = threadIdx.x; e < 2 * a.E + 1; e += WARPS * 32) sh[e] = 0;
    __syncthreads();
    // slots of each expert in all blocks and in the blocks before this one: every thread adds up some of the blocks' counts
    // of one expert
    const int groups = max(1, WARPS * 32 / a.E);
    for (int i = threadIdx.x; i < groups * a.E; i += WARPS * 32) {
        const int e = i % a.E;
        int all = 0, mine = 0;
#pragma unroll 4
        for (int b = i / a.E; b < (int)gridDim.x; b += groups) {
            const int c = __ldg(a.counts + (long)b * a.E + e);
            all += c;
            mine += b < (int)blockIdx.x ? c : 0;
        }
        atomicAdd(total + e, all);
        atomicAdd(before + e, mine);
    }
    __syncthreads();
    exclusive_sum(total, a.E);
    for (int e = threadIdx.x; e < a.E; e += WARPS * 32) before[e] += total[e];
    if (blockIdx.x == 0)
        for (int e = threadIdx.x; e <= a.E; e += WARPS * 32) a.offsets[e] = total[e];
    __syncthreads();
    const long i0 = (long)blockIdx.x * a.per_block * a.k, i1 = min((long)a.T * a.k, i0 + (long)a.per_block * a.k);
    place_slots<WARPS>(a, i0, i1, before, warp_count);
    clear_tail(a, total[a.E], (long)blockIdx.x * WARPS * 32 + threadIdx.x, (long)gridDim.x * WARPS * 32);
}

template <int G, int EPL, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) route_one_block_kernel(const RouteArgs a) {
    extern __shared__ int sh[];
    int *total = sh, *warp_count = sh + a.E + 1;
    for (int e = threadIdx.x; e < a.E; e += WARPS * 32) total[e] = 0;
    __syncthreads();
    rank_tokens<G, EPL, WARPS>(a, 0, a.T, total);
    __syncthreads();
    exclusive_sum(total, a.E);
    for (int e = threadIdx.x; e <= a.E; e += WARPS * 32) a.offsets[e] = total[e];
    place_slots<WARPS>(a, 0, (long)a.T * a.k, total, warp_count);
    clear_tail(a, total[a.E], threadIdx.x, WARPS * 32);
}

// dmu_s_j = sum_i J_ij dmu_g_i, dvar_s_j = sum_i J_ij^2 dvar_g_i over the chosen, J_ij = g_i (d_ij - g_j). G lanes per token,
// as in the forward pass; a warp writes zeros along the whole rows of its tokens, then the chosen experts' entries.
// VEC: rows of a multiple of four, 16-byte aligned.
constexpr int BWD_WARPS = 8;
template <int G, bool VEC>
__global__ void __launch_bounds__(BWD_WARPS * 32) route_bwd_kernel(int T, int E, int k, const int *__restrict__ expert,
                                                                   const float *__restrict__ mu_g, const float *__restrict__ dmu_g,
                                                                   const float *__restrict__ dvar_g, float *dmu_s, float *dvar_s) {
    constexpr int TOKENS = 32 / G;
    const long t0 = ((long)blockIdx.x * BWD_WARPS + (threadIdx.x >> 5)) * TOKENS;
    if (t0 >= T) return;
    const int lane = threadIdx.x & 31, l = lane & (G - 1);
    const long t = t0 + lane / G;
    int e = t < T && l < k ? __ldg(expert + t * k + l) : -1;
    if (e >= E) e = -1;
    const bool has = e >= 0;   // a slot without an expert has no part in the sums, whatever its deltas hold
    const float g = has ? __ldg(mu_g + t * k + l) : 0.f, d = has ? __ldg(dmu_g + t * k + l) : 0.f,
                w = has ? __ldg(dvar_g + t * k + l) : 0.f;
    float *m = dmu_s + t0 * E, *v = dvar_s + t0 * E;
    const int n = (int)min((long)TOKENS, T - t0) * E;
    if (VEC) {
        for (int c = lane * 4; c < n; c += 128) {
            *reinterpret_cast<float4 *>(m + c) = make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4 *>(v + c) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    } else {
        for (int c = lane; c < n; c += 32) m[c] = v[c] = 0.f;
    }
    float rest = 0.f, dm = 0.f, dv = 0.f;
    for (int i = 0; i < k; i++) {
        const float gi = __shfl_sync(FULL, g, i, G), di = __shfl_sync(FULL, d, i, G), wi = __shfl_sync(FULL, w, i, G);
        if (i != l) rest += gi, dm += gi * (d - di), dv += gi * gi * wi;
    }
    __syncwarp();   // the zeros lie below
    if (has) {
        dmu_s[t * E + e] = g * dm;
        dvar_s[t * E + e] = g * g * (rest * rest * w + dv);
    }
}

inline int launched(const char *what) {
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? TAGI_OK : cuda_fail(e, what);
}

// Tokens of a block: no more blocks than SMs, so that the second kernel's sum over the blocks before its own stays short,
// and no fewer than 32 tokens in one.
int per_block(int T) {
    const int p = (T + MAX_BLOCKS - 1) / MAX_BLOCKS;
    return p < 32 ? 32 : p;
}
int blocks_of(int T) { return (T + per_block(T) - 1) / per_block(T); }

template <int G, int EPL>
int route_launch(const RouteArgs &a, cudaStream_t st) {
    constexpr int WARPS = warps_for(G * EPL);
    const size_t ints = sizeof(int);
    if (a.T <= ONE_BLOCK_TOKENS) {
        route_one_block_kernel<G, EPL, WARPS><<<1, WARPS * 32, (a.E + 1 + WARPS * a.E) * ints, st>>>(a);
        return launched("route_one_block_kernel launch");
    }
    const int blocks = blocks_of(a.T);
    route_rank_kernel<G, EPL, WARPS><<<blocks, WARPS * 32, a.E * ints, st>>>(a);
    int rc = launched("route_rank_kernel launch");
    if (rc != TAGI_OK) return rc;
    route_place_kernel<WARPS><<<blocks, WARPS * 32, (2 * a.E + 1 + WARPS * a.E) * ints, st>>>(a);
    return launched("route_place_kernel launch");
}

int check_route(const char *who, int T, int E, int k) {
    if (T < 0 || E < 1 || E > MAX_EXPERTS) return fail(TAGI_ERR_INVALID_ARGUMENT, std::string(who) + ": 1 to 1024 experts, tokens must not be negative");
    if (k < 1 || k > E || k > MAX_K) return fail(TAGI_ERR_INVALID_ARGUMENT, std::string(who) + ": k must be 1 to 32 and at most the number of experts");
    if (T > MAX_TOKENS) return fail(TAGI_ERR_INVALID_ARGUMENT, std::string(who) + ": more than 2^30 tokens");
    if ((long)T * k >= (1L << 31)) return fail(TAGI_ERR_INVALID_ARGUMENT, std::string(who) + ": more than 2^31 slots");
    return TAGI_OK;
}

}  // namespace
}  // namespace tagi

using namespace tagi;

#define TAGI_PTR(p) TAGI_REQUIRE((p) != nullptr && aligned4(p), #p " is null or not 4-byte aligned")

extern "C" {

size_t tagi_route_workspace_bytes(int T, int E, int k) {
    if (T <= ONE_BLOCK_TOKENS || T > MAX_TOKENS || E < 1 || E > MAX_EXPERTS || k < 1 || k > E || k > MAX_K) return 0;
    return (size_t)blocks_of(T) * E * sizeof(int);
}

int tagi_route_fwd(int T, int E, int k, const float *mu_s, const float *var_s, int *expert, float *mu_g, float *var_g,
                   int *offsets, int *token, int *pos, void *workspace, size_t workspace_bytes, void *stream) {
    int rc = check_route(__func__, T, E, k);
    if (rc != TAGI_OK) return rc;
    TAGI_PTR(offsets);
    if (T > 0) {
        TAGI_PTR(mu_s);
        TAGI_REQUIRE(var_s == nullptr || aligned4(var_s), "var_s is not 4-byte aligned");
        TAGI_PTR(expert);
        TAGI_PTR(mu_g);
        TAGI_PTR(var_g);
        TAGI_PTR(token);
        TAGI_PTR(pos);
    }
    const size_t need = tagi_route_workspace_bytes(T, E, k);
    TAGI_REQUIRE(need == 0 || (workspace != nullptr && aligned4(workspace) && workspace_bytes >= need),
                 "workspace is null, not 4-byte aligned or smaller than tagi_route_workspace_bytes");
    const RouteArgs a{T, E, k, per_block(T), mu_s, var_s, expert, mu_g, var_g, offsets, token, pos, static_cast<int *>(workspace),
                      E % 4 == 0 && aligned16(mu_s)};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // the smallest group that has a lane for each slot and at most 16 scores a lane (what 32 warps have registers for)
    if (k <= 8 && E <= 32) return route_launch<8, 4>(a, st);
    if (k <= 8 && E <= 64) return route_launch<8, 8>(a, st);
    if (k <= 8 && E <= 128) return route_launch<8, 16>(a, st);
    if (k <= 16 && E <= 64) return route_launch<16, 4>(a, st);
    if (k <= 16 && E <= 128) return route_launch<16, 8>(a, st);
    if (k <= 16 && E <= 256) return route_launch<16, 16>(a, st);
    if (E <= 128) return route_launch<32, 4>(a, st);
    if (E <= 256) return route_launch<32, 8>(a, st);
    if (E <= 512) return route_launch<32, 16>(a, st);
    return route_launch<32, 32>(a, st);
}

int tagi_route_bwd(int T, int E, int k, const int *expert, const float *mu_g, const float *dmu_g, const float *dvar_g,
                   float *dmu_s, float *dvar_s, void *stream) {
    int rc = check_route(__func__, T, E, k);
    if (rc != TAGI_OK || T == 0) return rc;
    TAGI_PTR(expert);
    TAGI_PTR(mu_g);
    TAGI_PTR(dmu_g);
    TAGI_PTR(dvar_g);
    TAGI_PTR(dmu_s);
    TAGI_PTR(dvar_s);
    const bool vec = E % 4 == 0 && aligned16(dmu_s) && aligned16(dvar_s);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto start = [&](auto lanes) {
        constexpr int G = decltype(lanes)::value, TOKENS = BWD_WARPS * 32 / G;
        const int blocks = (T + TOKENS - 1) / TOKENS;
        if (vec) route_bwd_kernel<G, true><<<blocks, BWD_WARPS * 32, 0, st>>>(T, E, k, expert, mu_g, dmu_g, dvar_g, dmu_s, dvar_s);
        else route_bwd_kernel<G, false><<<blocks, BWD_WARPS * 32, 0, st>>>(T, E, k, expert, mu_g, dmu_g, dvar_g, dmu_s, dvar_s);
    };
    if (k <= 8) start(std::integral_constant<int, 8>());
    else if (k <= 16) start(std::integral_constant<int, 16>());
    else start(std::integral_constant<int, 32>());
    return launched("route_bwd_kernel launch");
}

}  // extern "C"
