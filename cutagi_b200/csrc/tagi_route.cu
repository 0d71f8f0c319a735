// Routing of tokens to experts: the k best experts of every token by the means of the router's scores, the moments of the
// softmax over the chosen scores (the gates), and the dispatch order, a stable counting sort of the token's slots by expert.
// The backward pass takes deltas of the gates to deltas of the scores.
//
// One warp ranks one token: each lane keeps E / 32 scores as order-preserving integers, and a warp-wide integer maximum
// followed by a warp-wide minimum of the indices that reach it gives the best expert, ties to the lowest index.
// The counting sort cuts the tokens into blocks. The first kernel also counts its block's slots per expert; the second
// adds up the counts of the blocks before its own and ranks its slots with warp matches. Nothing depends on the order in
// which warps run: shared-memory atomics only add integers. Up to ONE_BLOCK_TOKENS tokens both halves are one launch of
// one block.
#include "tagi_common.h"

#include <climits>

namespace tagi {
namespace {

constexpr int MAX_EXPERTS = 1024, MAX_K = 32;
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
};

// Order-preserving integer of a score; 0 for the scores that bar an expert (-inf, NaN). -0 counts as 0.
__device__ __forceinline__ unsigned score_key(float s) {
    if (!(s > -INFINITY)) return 0u;
    const unsigned u = __float_as_uint(s + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_score(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

// The warp's scores of token t, EPL to a lane
template <int EPL>
__device__ __forceinline__ void load_scores(const RouteArgs &a, long t, float (&score)[EPL]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int q = 0; q < EPL; q++) score[q] = q * 32 + lane < a.E ? __ldg(a.mu_s + t * a.E + q * 32 + lane) : -INFINITY;
}

// The whole warp ranks token t and writes its slots' experts and gates. Returns the expert of the lane's slot, or -1.
template <int EPL>
__device__ __forceinline__ int rank_token(const RouteArgs &a, long t, const float (&scores)[EPL]) {
    const int lane = threadIdx.x & 31;
    unsigned key[EPL];
#pragma unroll
    for (int q = 0; q < EPL; q++) key[q] = score_key(scores[q]);
    int mine = -1;        // slot `lane`: its expert and score
    float score = -INFINITY;
    for (int j = 0; j < a.k; j++) {
        unsigned best = 0;
#pragma unroll
        for (int q = 0; q < EPL; q++) best = max(best, key[q]);
        best = __reduce_max_sync(FULL, best);
        if (best == 0u) break;  // the experts left are barred
        unsigned at = UINT_MAX;
#pragma unroll
        for (int q = EPL - 1; q >= 0; q--)
            if (key[q] == best) at = q * 32 + lane;
        at = __reduce_min_sync(FULL, at);
#pragma unroll
        for (int q = 0; q < EPL; q++)
            if ((unsigned)(q * 32 + lane) == at) key[q] = 0u;
        if (lane == j) mine = (int)at, score = key_score(best);
    }
    // softmax over the chosen scores (slot 0 holds the largest); equal infinite scores share evenly
    const float top = __shfl_sync(FULL, score, 0);
    const float p = mine < 0 ? 0.f : score == top ? 1.f : expf(score - top);
    float z = p;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(FULL, z, o);
    const float g = mine < 0 ? 0.f : p / z;
    const float v = mine < 0 || a.var_s == nullptr ? 0.f : __ldg(a.var_s + t * a.E + mine);
    // var_g_i = g_i^2 ((1 - g_i)^2 v_i + sum_{j != i} g_j^2 v_j); 1 - g_i as the sum of the others does not cancel
    float rest = 0.f, others = 0.f;
    for (int j = 0; j < a.k; j++) {
        const float gj = __shfl_sync(FULL, g, j), vj = __shfl_sync(FULL, v, j);
        if (j != lane) rest += gj, others += gj * gj * vj;
    }
    if (lane < a.k) {
        const long i = t * a.k + lane;
        a.expert[i] = mine;
        a.mu_g[i] = g;
        a.var_g[i] = g * g * (rest * rest * v + others);
    }
    return mine;
}

// Ranks the tokens [t0, t1) of the block and adds their slots to count[e]. The next token's scores are on their way meanwhile.
template <int EPL, int WARPS>
__device__ __forceinline__ void rank_tokens(const RouteArgs &a, long t0, long t1, int *count) {
    long t = t0 + (threadIdx.x >> 5);
    float now[EPL], next[EPL];
    if (t < t1) load_scores<EPL>(a, t, now);
    for (; t < t1; t += WARPS) {
        if (t + WARPS < t1) load_scores<EPL>(a, t + WARPS, next);
        const int e = rank_token<EPL>(a, t, now);
        if (e >= 0) atomicAdd(count + e, 1);
#pragma unroll
        for (int q = 0; q < EPL; q++) now[q] = next[q];
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
            if (p >= 0) a.token[p] = (int)((i + lane) / a.k);
        }
    }
}

// slots without an expert leave the end of `token` empty
__device__ __forceinline__ void clear_tail(const RouteArgs &a, long live, long first, long stride) {
    for (long i = live + first; i < (long)a.T * a.k; i += stride) a.token[i] = -1;
}

template <int EPL, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) route_rank_kernel(const RouteArgs a) {
    extern __shared__ int count[];
    const long t0 = (long)blockIdx.x * a.per_block, t1 = min((long)a.T, t0 + a.per_block);
    for (int e = threadIdx.x; e < a.E; e += WARPS * 32) count[e] = 0;
    __syncthreads();
    rank_tokens<EPL, WARPS>(a, t0, t1, count);
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

template <int EPL, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) route_one_block_kernel(const RouteArgs a) {
    extern __shared__ int sh[];
    int *total = sh, *warp_count = sh + a.E + 1;
    for (int e = threadIdx.x; e < a.E; e += WARPS * 32) total[e] = 0;
    __syncthreads();
    rank_tokens<EPL, WARPS>(a, 0, a.T, total);
    __syncthreads();
    exclusive_sum(total, a.E);
    for (int e = threadIdx.x; e <= a.E; e += WARPS * 32) a.offsets[e] = total[e];
    place_slots<WARPS>(a, 0, (long)a.T * a.k, total, warp_count);
    clear_tail(a, total[a.E], threadIdx.x, WARPS * 32);
}

// dmu_s_j = sum_i J_ij dmu_g_i, dvar_s_j = sum_i J_ij^2 dvar_g_i over the chosen, J_ij = g_i (d_ij - g_j); one warp per token
// writes zeros along the whole row, then the chosen experts' entries. VEC: rows of a multiple of four, 16-byte aligned.
constexpr int BWD_WARPS = 8;
template <bool VEC>
__global__ void __launch_bounds__(BWD_WARPS * 32) route_bwd_kernel(int T, int E, int k, const int *__restrict__ expert,
                                                                   const float *__restrict__ mu_g, const float *__restrict__ dmu_g,
                                                                   const float *__restrict__ dvar_g, float *dmu_s, float *dvar_s) {
    const long t = (long)blockIdx.x * BWD_WARPS + (threadIdx.x >> 5);
    if (t >= T) return;
    const int lane = threadIdx.x & 31;
    int e = lane < k ? __ldg(expert + t * k + lane) : -1;
    if (e >= E) e = -1;
    const bool has = e >= 0;   // a slot without an expert has no part in the sums, whatever its deltas hold
    const float g = has ? __ldg(mu_g + t * k + lane) : 0.f, d = has ? __ldg(dmu_g + t * k + lane) : 0.f,
                w = has ? __ldg(dvar_g + t * k + lane) : 0.f;
    if (VEC) {
        for (int c = lane * 4; c < E; c += 128) {
            *reinterpret_cast<float4 *>(dmu_s + t * E + c) = make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4 *>(dvar_s + t * E + c) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    } else {
        for (int c = lane; c < E; c += 32) dmu_s[t * E + c] = dvar_s[t * E + c] = 0.f;
    }
    float rest = 0.f, dm = 0.f, dv = 0.f;
    for (int i = 0; i < k; i++) {
        const float gi = __shfl_sync(FULL, g, i), di = __shfl_sync(FULL, d, i), wi = __shfl_sync(FULL, w, i);
        if (i != lane) rest += gi, dm += gi * (d - di), dv += gi * gi * wi;
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

template <int EPL>
int route_launch(const RouteArgs &a, cudaStream_t st) {
    constexpr int WARPS = warps_for(EPL * 32);
    const size_t ints = sizeof(int);
    if (a.T <= ONE_BLOCK_TOKENS) {
        route_one_block_kernel<EPL, WARPS><<<1, WARPS * 32, (a.E + 1 + WARPS * a.E) * ints, st>>>(a);
        return launched("route_one_block_kernel launch");
    }
    const int blocks = blocks_of(a.T);
    route_rank_kernel<EPL, WARPS><<<blocks, WARPS * 32, a.E * ints, st>>>(a);
    int rc = launched("route_rank_kernel launch");
    if (rc != TAGI_OK) return rc;
    route_place_kernel<WARPS><<<blocks, WARPS * 32, (2 * a.E + 1 + WARPS * a.E) * ints, st>>>(a);
    return launched("route_place_kernel launch");
}

int check_route(const char *who, int T, int E, int k) {
    if (T < 0 || E < 1 || E > MAX_EXPERTS) return fail(TAGI_ERR_INVALID_ARGUMENT, std::string(who) + ": 1 to 1024 experts, tokens must not be negative");
    if (k < 1 || k > E || k > MAX_K) return fail(TAGI_ERR_INVALID_ARGUMENT, std::string(who) + ": k must be 1 to 32 and at most the number of experts");
    if ((long)T * k >= (1L << 31)) return fail(TAGI_ERR_INVALID_ARGUMENT, std::string(who) + ": more than 2^31 slots");
    return TAGI_OK;
}

}  // namespace
}  // namespace tagi

using namespace tagi;

#define TAGI_PTR(p) TAGI_REQUIRE((p) != nullptr && aligned4(p), #p " is null or not 4-byte aligned")

extern "C" {

size_t tagi_route_workspace_bytes(int T, int E, int k) {
    if (T <= ONE_BLOCK_TOKENS || E < 1 || E > MAX_EXPERTS || k < 1 || k > E || k > MAX_K) return 0;
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
    const RouteArgs a{T, E, k, per_block(T), mu_s, var_s, expert, mu_g, var_g, offsets, token, pos, static_cast<int *>(workspace)};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (E <= 32) return route_launch<1>(a, st);
    if (E <= 128) return route_launch<4>(a, st);
    if (E <= 256) return route_launch<8>(a, st);
    if (E <= 512) return route_launch<16>(a, st);
    return route_launch<32>(a, st);
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
    const int blocks = (T + BWD_WARPS - 1) / BWD_WARPS;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (E % 4 == 0 && aligned16(dmu_s) && aligned16(dvar_s))
        route_bwd_kernel<true><<<blocks, BWD_WARPS * 32, 0, st>>>(T, E, k, expert, mu_g, dmu_g, dvar_g, dmu_s, dvar_s);
    else
        route_bwd_kernel<false><<<blocks, BWD_WARPS * 32, 0, st>>>(T, E, k, expert, mu_g, dmu_g, dvar_g, dmu_s, dvar_s);
    return launched("route_bwd_kernel launch");
}

}  // extern "C"
