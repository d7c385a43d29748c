// What the two paged-attention kernels (short queries, paged_attention.cu; chunks, paged_attention_chunk.cu) share: the
// parameters, how the work is cut into units, and how partial results of a split item are joined.
//
// Work.  An ITEM is (request, tile of query rows, key head): the rows are the request's queries times the query heads of
// that key head (token-major), so that all of them share the keys.  An item is as many UNITS as it has blocks of
// UNIT visible keys, at least one, and weighs `cost` units more, for what its beginning and end take.  All items are laid end
// to end (requests, then tiles, then heads) and every CTA of the grid takes an equal, contiguous stretch of that weight:
// whatever the lengths, the CTAs finish together, and nothing but the lengths on the device decides it (a captured launch
// replays with new lengths).  A stretch boundary inside an item's units splits it (one inside its cost moves to its
// beginning); short items are never split.  Each part leaves its unnormalised sum, its maximum and its weight in the workspace, and the CTA that arrives
// last (a counter in the workspace) joins them in the order of the keys -- so results do not depend on who was last.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "kv_cache.cuh"
#include "math.cuh"
#include "ptx_sm100.cuh"

namespace b200 {

struct PagedParams {
    const void* q;
    void* out;
    float* lse;
    const float* k_scale;
    const float* v_scale;
    const int* table;
    const int* starts;
    const int* lens;
    size_t q_stride, out_stride;
    int requests, group, kv_heads, max_query, max_blocks, num_blocks, block_size, shift;
    int rows;                       // of q and out
    int rows_above, rows_upto;      // this launch takes the requests with rows_above < queries * group <= rows_upto
    float scale_log2;               // softmax scale * log2(e)
    int causal;
    int cost, unsplit;              // weight of an item beside its units; items of up to so many units stay whole where the launch has none larger
    int* counters;                  // [CTAs], zero between calls
    float* partials;                // [CTAs][2][tile rows * (head_dim + 2)]: sums, maxima, weights
    int* status;
};

struct PagedRequest { int start, full, n, len, rows; };

__device__ __forceinline__ PagedRequest paged_request(const PagedParams& p, int r) {
    PagedRequest q;
    q.start = __ldg(p.starts + r);
    q.full = max(0, __ldg(p.starts + r + 1) - q.start);
    q.n = q.start < 0 ? 0 : max(0, min(min(q.full, p.max_query), p.rows - q.start));
    q.len = static_cast<int>(min(static_cast<long long>(max(0, __ldg(p.lens + r))), static_cast<long long>(p.max_blocks) << p.shift));
    const long long rows = static_cast<long long>(q.n) * p.group;
    q.rows = rows > p.rows_above && rows <= p.rows_upto ? static_cast<int>(rows) : 0;
    return q;
}
// Number of keys that query i of the request sees.
__device__ __forceinline__ int paged_limit(const PagedParams& p, const PagedRequest& q, int i) {
    return p.causal ? min(q.len, max(0, q.len - q.full + i + 1)) : q.len;
}
// Keys that some row of tile t (TILE rows) sees: those of its last query.
template <int TILE>
__device__ __forceinline__ int paged_tile_end(const PagedParams& p, const PagedRequest& q, int t) {
    return paged_limit(p, q, (min((t + 1) * TILE, q.rows) - 1) / p.group);
}
template <int TILE, int UNIT>
__device__ __forceinline__ int paged_tile_units(const PagedParams& p, const PagedRequest& q, int t) {
    return max(1, (paged_tile_end<TILE>(p, q, t) + UNIT - 1) / UNIT);
}
// Weight of a request's items of ONE key head.
template <int TILE, int UNIT>
__device__ __forceinline__ long long paged_request_weight(const PagedParams& p, const PagedRequest& q) {
    long long n = 0;
    for (int t = 0; t * TILE < q.rows; ++t) n += paged_tile_units<TILE, UNIT>(p, q, t) + p.cost;
    return n;
}

// How the launch's weight is shared out: the same for every thread of a CTA, kept in shared memory.
struct PagedShares {
    long long lo, total, share;     // this CTA's first position; all weight; weight per CTA (one more for the first `extra` CTAs)
    int ctas, extra;                // CTAs that have a stretch (never more than weight, so none is empty)
    int found_r;                    // request of the first position, and its beginning relative to lo
    long long found_at;
    long long sums[32];
    int most[32];
};
// Where a warp stands in the sequence of items.  Positions count from the CTA's first.
struct PagedCursor {
    int hi;                         // end of the CTA's stretch
    int item;                       // beginning of the current item (below 0 where another CTA has it)
    int r, t, h, units;             // current item and its number of units
    int cost;
    bool whole;                     // items are not split: one belongs to the CTA with its last position
    PagedRequest q;
    // the CTA's part of the item's units
    __device__ __forceinline__ int from() const { return whole ? 0 : max(0, -item - cost); }
    __device__ __forceinline__ int to() const { return whole ? (item + cost + units <= hi ? units : 0) : min(units, hi - item - cost); }
};

// Sums all requests' weights (every CTA for itself: 12 bytes per request out of L2) and finds the item where the CTA's
// stretch begins.  False when the CTA has nothing to do.
template <int THREADS, int TILE, int UNIT>
__device__ __forceinline__ bool paged_begin(const PagedParams& p, PagedCursor& c, PagedShares& sh) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int per = (p.requests + THREADS - 1) / THREADS;
    const int r0 = min(static_cast<int>(threadIdx.x) * per, p.requests), r1 = min(r0 + per, p.requests);
    long long mine = 0;
    int most = 0;
    for (int r = r0; r < r1; ++r) {
        const PagedRequest q = paged_request(p, r);
        mine += paged_request_weight<TILE, UNIT>(p, q);
        if (q.rows > 0) most = max(most, (q.len + UNIT - 1) / UNIT);
    }
    mine *= p.kv_heads;
    long long upto = mine;
    most = __reduce_max_sync(0xffffffffu, most);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const long long x = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += x; }
    if (lane == 31) { sh.sums[w] = upto; sh.most[w] = most; }
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) { const long long x = sh.sums[i]; total += x; if (i < w) before += x; most = max(most, sh.most[i]); }
    c.whole = most <= p.unsplit;
    c.cost = p.cost;
    upto += before;
    if (total == 0) return false;
    if (total > static_cast<long long>(gridDim.x) << 30) {         // positions within a stretch are ints: months of work, refused
        if (threadIdx.x == 0) atomicCAS(p.status, ST_OK, ST_WAIT_TIMEOUT | (0x6f << 8));
        return false;
    }
    const int ctas = static_cast<int>(min(static_cast<long long>(gridDim.x), total));
    if (static_cast<int>(blockIdx.x) >= ctas) return false;
    const long long share = total / ctas;
    const int extra = static_cast<int>(total - share * ctas);
    const long long lo = share * blockIdx.x + min(static_cast<int>(blockIdx.x), extra);
    c.hi = static_cast<int>(share) + (static_cast<int>(blockIdx.x) < extra ? 1 : 0);
    if (upto - mine <= lo && lo < upto) {
        long long at = upto - mine;
        int r = r0;
        for (;; ++r) {
            const long long n = paged_request_weight<TILE, UNIT>(p, paged_request(p, r)) * p.kv_heads;
            if (lo < at + n) break;
            at += n;
        }
        sh.lo = lo; sh.total = total; sh.share = share; sh.ctas = ctas; sh.extra = extra;
        sh.found_r = r; sh.found_at = at - lo;
    }
    __syncthreads();
    long long at = sh.found_at;
    c.r = sh.found_r;
    c.q = paged_request(p, c.r);
    for (c.t = 0;; ++c.t) {
        c.units = paged_tile_units<TILE, UNIT>(p, c.q, c.t);
        const long long heads = static_cast<long long>(c.units + p.cost) * p.kv_heads;
        if (at + heads > 0) break;
        at += heads;
    }
    c.h = static_cast<int>(-at / (c.units + p.cost));
    c.item = static_cast<int>(at + static_cast<long long>(c.h) * (c.units + p.cost));
    return c.to() > 0;
}
// To the CTA's next item; false, and the cursor as it was, when its stretch has no part of it.
template <int TILE, int UNIT>
__device__ __forceinline__ bool paged_next(const PagedParams& p, PagedCursor& c) {
    const int item = c.item + c.units + p.cost;
    if (item + p.cost >= c.hi) return false;                   // also where there is no further request
    PagedCursor n = c;
    n.item = item;
    if (++n.h == p.kv_heads) {
        n.h = 0;
        ++n.t;
        while (n.t * TILE >= n.q.rows) { n.t = 0; ++n.r; n.q = paged_request(p, n.r); }
        n.units = paged_tile_units<TILE, UNIT>(p, n.q, n.t);
    }
    if (n.to() <= 0) return false;
    c = n;
    return true;
}
// CTA whose stretch holds position u (of the launch).
__device__ __forceinline__ int paged_cta_of(const PagedShares& s, long long u) {
    const long long big = (s.share + 1) * s.extra;                 // of the CTAs that have one more
    return u < big ? static_cast<int>(u / (s.share + 1)) : s.extra + static_cast<int>((u - big) / s.share);
}

// CTAs with the item's first and last unit.
__device__ __forceinline__ int paged_first(const PagedShares& s, const PagedCursor& c) { return paged_cta_of(s, s.lo + c.item + c.cost); }
__device__ __forceinline__ int paged_last(const PagedShares& s, const PagedCursor& c) { return paged_cta_of(s, s.lo + c.item + c.cost + c.units - 1); }

__device__ __forceinline__ float paged_clamp_scale(float s) { return fminf(fmaxf(s, 0x1p-40f), 0x1p72f); }

template <typename T> __device__ __forceinline__ uint32_t paged_pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t paged_pack2<__nv_bfloat16>(float a, float b) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
template <> __device__ __forceinline__ uint32_t paged_pack2<__half>(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }

// Result of row `row` of the item from its sums `o` (values d .. d + N - 1), weight `l` and reference maximum `m` (log2 units).
template <typename T, int D, int N>
__device__ __forceinline__ void paged_finish(const PagedParams& p, const PagedCursor& c, int row, int d, const float (&o)[N], float m, float l) {
    const int token = row / p.group, head = c.h * p.group + (row - token * p.group);
    const size_t at = static_cast<size_t>(c.q.start) + token;
    const bool none = l == 0.0f;                                   // no key seen: zero and -inf
    const float inv = none ? 0.0f : 1.0f / l;
    T* dst = static_cast<T*>(p.out) + at * p.out_stride + static_cast<size_t>(head) * D + d;
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N; i += 2) w[i / 2] = paged_pack2<T>(none ? 0.0f : o[i] * inv, none ? 0.0f : o[i + 1] * inv);
    if constexpr (N == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (N == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    else {
#pragma unroll
        for (int i = 0; i < N; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = w[i / 2];
    }
    if (p.lse && d == 0) p.lse[at * (static_cast<size_t>(p.group) * p.kv_heads) + head] = none ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

// The parts of split items that this CTA computed (at most two: the item that its stretch begins in and the one that it
// ends in) have left their sums in its slots.  At the end of its stretch it announces them and joins the items of which all
// parts are there now.  Announcing late costs nothing -- somebody has to be last -- and keeps the fence and the round trip
// of the counters out of the way of the copies.  flags: 2 ints of shared memory.
template <typename T, int D, int THREADS, int TILE>
__device__ __forceinline__ void paged_join(const PagedParams& p, const PagedShares& sh, const PagedCursor& c) {
    const int first = paged_first(sh, c), parts = paged_last(sh, c) - first + 1;
    constexpr size_t SLOT = static_cast<size_t>(TILE) * (D + 2);
    auto slot = [&](int i) { return p.partials + (static_cast<size_t>(first + i) * 2 + (i == 0 ? 1 : 0)) * SLOT; };
    // One warp per row; lane i has the maxima and weights of parts i, i + 32, .. (there can be hundreds) and the values D / 32 i .. of
    // the sums, of which it asks for BATCH parts at once: 16 took 107 us for 64 requests of 8000 keys | 61 us for one of 131 K,
    // 8 105 | 61, 4 104 | 60.
    constexpr int VPL = D / 32, BATCH = 4;
    const int lane = threadIdx.x & 31, rows = min(TILE, c.q.rows - c.t * TILE);
    for (int row = threadIdx.x >> 5; row < rows; row += THREADS / 32) {
        float mi, li, o[VPL], v[BATCH][VPL];
        auto weights = [&](int i0) {         // of parts i0 + lane
            const float* ml = slot(min(i0 + lane, parts - 1)) + TILE * D + row;
            mi = __ldcg(ml); li = __ldcg(ml + TILE);
            if (i0 + lane >= parts) { mi = -INFINITY; li = 0.0f; }
        };
        auto sums = [&](int i) {             // of parts i .. i + BATCH - 1 (beyond the last: the last's)
#pragma unroll
            for (int y = 0; y < BATCH; ++y) {
                const float* src = slot(min(i + y, parts - 1)) + row * D + lane * VPL;
                if constexpr (VPL == 4) { const float4 u = __ldcg(reinterpret_cast<const float4*>(src)); v[y][0] = u.x; v[y][1] = u.y; v[y][2] = u.z; v[y][3] = u.w; }
                else { const float2 u = __ldcg(reinterpret_cast<const float2*>(src)); v[y][0] = u.x; v[y][1] = u.y; }
            }
        };
        weights(0);
        sums(0);
        float m = mi, l = 0.0f;
        for (int i = lane + 32; i < parts; i += 32) m = fmaxf(m, __ldcg(slot(i) + TILE * D + row));
#pragma unroll
        for (int y = 16; y > 0; y >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, y));
        if (m == -INFINITY) m = 0.0f;
#pragma unroll
        for (int y = 0; y < VPL; ++y) o[y] = 0.0f;
#pragma unroll 1
        for (int i0 = 0; i0 < parts; i0 += BATCH) {
            if (i0 > 0) {
                if (i0 % 32 == 0) weights(i0);
                sums(i0);
            }
            if (i0 % 32 == 0) { mi = ex2_approx(mi - m); l = fmaf(mi, li, l); }      // now the factors
#pragma unroll
            for (int y = 0; y < BATCH; ++y) {
                const float w = __shfl_sync(0xffffffffu, mi, (i0 + y) & 31);
                if (i0 + y < parts)
#pragma unroll
                    for (int e = 0; e < VPL; ++e) o[e] = fmaf(v[y][e], w, o[e]);
            }
        }
#pragma unroll
        for (int y = 16; y > 0; y >>= 1) l += __shfl_xor_sync(0xffffffffu, l, y);
        paged_finish<T, D>(p, c, c.t * TILE + row, lane * VPL, o, m, l);
    }
}

// The same for the large tiles of chunks, which are split in two or three: a thread has one row, and eight values of it at a time.  The
// sums lie four values of all rows after four values of all rows, so that a warp stores and reads 512 bytes in a piece.
template <typename T, int D, int THREADS, int TILE>
__device__ __forceinline__ void paged_join_tile(const PagedParams& p, const PagedShares& sh, const PagedCursor& c) {
    const int first = paged_first(sh, c), parts = paged_last(sh, c) - first + 1;
    constexpr size_t SLOT = static_cast<size_t>(TILE) * (D + 2);
    constexpr int STEP = THREADS / TILE, AT_ONCE = 4 * STEP <= D / 8 ? 4 : D / 8 / STEP;
    static_assert(THREADS % TILE == 0 && D / 8 % (STEP * AT_ONCE) == 0, "whole rows");
    const int in_tile = threadIdx.x % TILE, row = c.t * TILE + in_tile;
    if (row >= c.q.rows) return;
    auto slot = [&](int i) { return p.partials + (static_cast<size_t>(first + i) * 2 + (i == 0 ? 1 : 0)) * SLOT; };
    float m = -INFINITY, l = 0.0f;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) m = fmaxf(m, __ldcg(slot(i) + TILE * D + in_tile));
    if (m == -INFINITY) m = 0.0f;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) l = fmaf(ex2_approx(__ldcg(slot(i) + TILE * D + in_tile) - m), __ldcg(slot(i) + TILE * (D + 1) + in_tile), l);
#pragma unroll 1
    for (int g = threadIdx.x / TILE; g < D / 8; g += STEP * AT_ONCE) {
        float o[AT_ONCE][8] = {};
#pragma unroll 1
        for (int i = 0; i < parts; i += 2) {
            float w[2];
            float4 v[2][AT_ONCE][2];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const float* src = slot(min(i + y, parts - 1));
                w[y] = __ldcg(src + TILE * D + in_tile);
#pragma unroll
                for (int x = 0; x < AT_ONCE; ++x)
#pragma unroll
                    for (int z = 0; z < 2; ++z) v[y][x][z] = __ldcg(reinterpret_cast<const float4*>(src) + ((g + x * STEP) * 2 + z) * TILE + in_tile);
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                if (i + y >= parts) break;
                const float f = ex2_approx(w[y] - m);
#pragma unroll
                for (int x = 0; x < AT_ONCE; ++x)
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        o[x][z * 4] = fmaf(v[y][x][z].x, f, o[x][z * 4]); o[x][z * 4 + 1] = fmaf(v[y][x][z].y, f, o[x][z * 4 + 1]);
                        o[x][z * 4 + 2] = fmaf(v[y][x][z].z, f, o[x][z * 4 + 2]); o[x][z * 4 + 3] = fmaf(v[y][x][z].w, f, o[x][z * 4 + 3]);
                    }
            }
        }
#pragma unroll
        for (int x = 0; x < AT_ONCE; ++x) paged_finish<T, D>(p, c, row, (g + x * STEP) * 8, o[x], m, l);
    }
}

template <typename T, int D, int THREADS, int TILE>
__device__ __forceinline__ void paged_announce(const PagedParams& p, const PagedShares& sh, const PagedCursor (&split)[2], const int (&is_split)[2], int* flags) {
    __syncthreads();                                               // all sums are written, is_split and split are set
    if (!is_split[0] && !is_split[1]) return;
    if (threadIdx.x == 0) {
        __threadfence();                                           // the sums before the arrivals
        int first[2], parts[2], before[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            flags[i] = 0;
            if (!is_split[i]) continue;
            first[i] = paged_first(sh, split[i]);
            parts[i] = paged_last(sh, split[i]) - first[i] + 1;
            before[i] = atomicAdd(p.counters + first[i], 1);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (is_split[i] && before[i] == parts[i] - 1) { flags[i] = 1; p.counters[first[i]] = 0; }   // as the next call finds it
        __threadfence();                                           // the other parts' sums after their arrivals
    }
    __syncthreads();
    for (int i = 0; i < 2; ++i)
        if (flags[i]) {
            if constexpr (TILE >= 64) paged_join_tile<T, D, THREADS, TILE>(p, sh, split[i]);
            else paged_join<T, D, THREADS, TILE>(p, sh, split[i]);
        }
}

}  // namespace b200
