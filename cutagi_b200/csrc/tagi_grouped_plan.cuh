// How the tensor-core kernels of the Linear layers grouped by expert share out their tiles, and the kernel that joins the tiles
// that were cut.
//
// Items (a tile's mean or its variance) go round the workers (CTAs, or pairs of them): the two kinds of a tile are neighbours, so
// two workers fetch the same weights at the same time, and a worker's kinds alternate from one item to the next (in the forward
// pass a variance costs twice a mean). What is left when the rounds no longer fill the GPU is cut along the contraction, so that
// all workers get the same number of chunks: each has at most the end of one tile (LATER) and the beginning of another (BEGIN),
// whose sums go to the workspace, and grouped_join_kernel adds up and writes out the tiles that were cut.
#pragma once
#include "tagi_grouped.h"

namespace tagi {
namespace {

constexpr int MEAN = 0, VAR = 1;
constexpr int WHOLE = -1, LATER = 0, BEGIN = 1;   // an item's part

struct Plan {
    int items, whole;   // all items; those that go round
    int chunks;         // of the items that are cut; -1: not looked at yet
};
// forward: as many means as variances for each worker, so the rounds come in twos
__device__ __forceinline__ Plan make_plan(bool forward, int items, int workers, bool may_cut) {
    const int round = forward ? 2 * workers : workers;
    return Plan{items, may_cut ? items / round * round : items, may_cut ? -1 : 0};
}
__device__ __forceinline__ int kind_of(int i, int workers) { return (i + 2 * (i >> 1) / workers) & 1; }

// Whether the rest is cut: if that saves at least `saves` chunks, what joining the tiles costs. chunks_of(i): an item's. start: 2
// * workers + 1 entries of shared memory. Called by one whole warp, when the whole rounds have been handed out.
template <class F>
__device__ __forceinline__ void look_at_rest(int *start, int workers, int saves, Plan &p, F chunks_of) {
    const int lane = threadIdx.x & 31;
    int carry = 0, longest = 0;
    for (int j0 = 0; j0 < p.items - p.whole; j0 += 32) {
        const int j = j0 + lane, i = p.whole + j, mine = i < p.items ? chunks_of(i) : 0;
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += u;
        }
        if (i < p.items) start[j] = carry + sum - mine;
        longest = max(longest, __reduce_max_sync(0xffffffffu, mine));
        carry += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) start[p.items - p.whole] = carry;
    __syncwarp();
    // uncut, the last round takes as long as its longest item; two rounds (forward) as a variance and a mean
    const int uncut = p.items - p.whole > workers ? longest + longest / 2 : longest;
    const bool cut = uncut - (carry + workers - 1) / workers >= saves;
    p.chunks = cut ? carry : 0;
    if (!cut) p.whole = p.items;
}

// Item j of a worker: the item's number, and which of its chunks (chunks == 0: all).
struct Share {
    int i, from, chunks, part;
};
template <class F>
__device__ __forceinline__ bool share_of(int *start, Plan &p, int worker, int workers, int saves, int j, F chunks_of, Share &s) {
    s.i = worker + j * workers, s.from = s.chunks = 0, s.part = WHOLE;
    if (s.i >= p.whole && p.chunks < 0) look_at_rest(start, workers, saves, p, chunks_of);
    if (s.i < p.whole) return true;
    // this worker's chunks of the tiles that are cut, one tile after the other
    const int begin = (int)((long)p.chunks * worker / workers), end = (int)((long)p.chunks * (worker + 1) / workers), rest = p.items - p.whole;
    if (begin == end) return false;
    int lo = 0, hi = rest - 1;   // the tile of the first of them
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (start[mid] <= begin) lo = mid; else hi = mid - 1;
    }
    lo += j - p.whole / workers;
    if (lo >= rest || start[lo] >= end) return false;
    const int last = start[lo + 1], c0 = max(begin, start[lo]), c1 = min(end, last);
    s.i = p.whole + lo;
    s.from = c0 - start[lo];
    s.chunks = c1 - c0;
    s.part = s.from > 0 ? LATER : c1 < last ? BEGIN : WHOLE;
    return true;
}

// What a partial sum belongs to, for the kernel that joins them; `ends`: it holds the tile's last chunk.
struct Piece {
    int used, ends, e, m0, c0, cols, bn, kind;
};
// The workers' partial sums in the workspace, two each: [columns][features], and behind tiles of 256 features the sums of the
// deltas of their columns (parameter pass); then what they belong to.
template <int FEATURES, int WIDTH>
struct Parts {
    static constexpr int FLOATS = FEATURES * WIDTH, PITCH = FLOATS + (FEATURES == 256 ? WIDTH : 0);
    __device__ static float *of(const GroupedArgs &a, int worker, int part) { return a.parts + (size_t)(worker * 2 + part) * PITCH; }
    __device__ static Piece *piece(const GroupedArgs &a, int workers, int worker, int part) {
        return reinterpret_cast<Piece *>(a.parts + (size_t)workers * 2 * PITCH) + worker * 2 + part;
    }
    static constexpr size_t bytes(int workers) { return (size_t)workers * 2 * (PITCH * sizeof(float) + sizeof(Piece)); }
};

// Feature (of 128) at place p of an operand whose features are MIXED: place 4 i + c holds feature i + 32 c.
__device__ __forceinline__ int feature_at(bool mixed, int p) { return mixed ? (p & 3) * 32 + (p >> 2) : p; }

// Adds up the partial sums of the tiles that were cut, in the order of the contraction, and writes them out. blockIdx.x: a
// worker's partial sum that begins a tile, the others do nothing; blockIdx.y: eight columns of it. A thread has a feature.
constexpr int JOIN_COLUMNS = 8;
template <int PASS, int FEATURES, int WIDTH>
__global__ void __launch_bounds__(FEATURES) grouped_join_kernel(const GroupedArgs a, int workers, bool mixed) {
    using P = Parts<FEATURES, WIDTH>;
    const int worker = blockIdx.x, x0 = blockIdx.y * JOIN_COLUMNS;
    const Piece t = *P::piece(a, workers, worker, BEGIN);
    if (!t.used || x0 >= t.cols) return;
    float acc[JOIN_COLUMNS], bias = 0.f;
    const bool sum = PASS == PARAM && a.var_b && t.m0 == 0 && blockIdx.y == 0 && (int)threadIdx.x < t.cols;
#pragma unroll
    for (int x = 0; x < JOIN_COLUMNS; x++) acc[x] = 0.f;
    bool ends = false;
    for (int q = worker; q < workers && !ends; q++) {   // a tile that begins here goes on with the next workers
        const int part = q == worker ? BEGIN : LATER;
        const Piece *piece = P::piece(a, workers, q, part);
        if (!piece->used) continue;   // a worker without a chunk
        const float *p = P::of(a, q, part);
#pragma unroll
        for (int x = 0; x < JOIN_COLUMNS; x++)
            if (x0 + x < t.cols) acc[x] += p[(x0 + x) * FEATURES + threadIdx.x];
        if (sum) bias += p[P::FLOATS + threadIdx.x];
        ends = piece->ends;
    }
    if (sum) {
        const size_t o = (size_t)t.e * a.N + t.c0 + threadIdx.x;
        const float vb = __ldg(a.var_b + o);
        (t.kind == VAR ? a.ob1 : a.ob0)[o] = t.kind == VAR ? vb * vb * bias : vb * bias;
    }
    const int m = t.m0 + (threadIdx.x & ~127) + feature_at(mixed, threadIdx.x & 127), ld = PASS == FWD ? a.N : a.K;
    if (m >= ld) return;
    const size_t base = ((PASS == PARAM ? (size_t)t.e * a.N : 0) + t.c0 + x0) * ld + m;
    const float *scale = PASS == PARAM ? a.var_w : a.jcb;
    float add = 0.f;
    if (PASS == FWD && a.mu_b) add = __ldg((t.kind == VAR ? a.var_b : a.mu_b) + (size_t)t.e * a.N + m);
#pragma unroll
    for (int x = 0; x < JOIN_COLUMNS; x++) {
        if (x0 + x >= t.cols) break;
        const size_t o = base + (size_t)x * ld;
        float z = acc[x] + add;
        if (PASS != FWD && scale) {
            const float f = __ldg(scale + o);
            z = t.kind == VAR ? z * f * f : z * f;
        }
        (t.kind == VAR ? a.o1 : a.o0)[o] = z;
    }
}

}  // namespace
}  // namespace tagi
