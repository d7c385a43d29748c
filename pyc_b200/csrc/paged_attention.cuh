// What the two paged-attention kernels (short queries, paged_attention.cu; chunks, paged_attention_chunk.cu) share: the
// parameters, how the work is cut into units, and how partial results of a split item are joined.
//
// Work.  An ITEM is (request, tile of query rows, key head): the rows are the request's queries times the query heads of
// that key head (token-major), so that all of them share the keys.  An item is as many UNITS as it has blocks of
// kUnitKeys visible keys, at least one.  All items' units are laid end to end (requests, then tiles, then heads) and every
// CTA of the grid takes an equal, contiguous stretch: whatever the lengths, the CTAs finish together, and nothing but the
// lengths on the device decides it (a captured launch replays with new lengths).  A stretch boundary inside an item
// splits it; each part leaves its unnormalised sum, its maximum and its weight in the workspace, and the CTA that arrives
// last (a counter in the workspace) joins them in the order of the keys -- so results do not depend on who was last.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "kv_cache.cuh"
#include "math.cuh"

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
    int rows_above, rows_upto;      // this launch takes the requests with rows_above < queries * group <= rows_upto
    float scale_log2;               // softmax scale * log2(e)
    int causal;
    int* counters;                  // [CTAs], zero between calls
    float* partials;                // [CTAs][2][tile rows * (head_dim + 2)]
    int* status;
};

struct PagedRequest { int start, full, n, len, rows; };

__device__ __forceinline__ PagedRequest paged_request(const PagedParams& p, int r) {
    PagedRequest q;
    q.start = __ldg(p.starts + r);
    q.full = max(0, __ldg(p.starts + r + 1) - q.start);
    q.n = min(q.full, p.max_query);
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
// Units of a request for ONE key head.
template <int TILE, int UNIT>
__device__ __forceinline__ long long paged_request_units(const PagedParams& p, const PagedRequest& q) {
    long long n = 0;
    for (int t = 0; t * TILE < q.rows; ++t) n += paged_tile_units<TILE, UNIT>(p, q, t);
    return n;
}

// Where a CTA stands in the sequence of items; all threads of the CTA hold the same values.
struct PagedCursor {
    long long lo, hi;               // this CTA's stretch of units
    long long item;                 // first unit of the current item
    long long total;                // units of the launch
    int ctas;                       // CTAs that have a stretch (never more than units, so none is empty)
    int r, t, h, units;             // current item and its number of units
    PagedRequest q;
};

// Sums all requests' units (every CTA for itself: 12 bytes per request out of L2) and finds the item where the CTA's
// stretch begins.  False when the CTA has nothing to do.  `min_units`: no CTA gets fewer, so that short work is not cut
// into pieces that cost more to join than to compute.
template <int THREADS, int TILE, int UNIT>
__device__ __forceinline__ bool paged_begin(const PagedParams& p, PagedCursor& c, long long* scratch, int min_units) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int per = (p.requests + THREADS - 1) / THREADS;
    const int r0 = min(static_cast<int>(threadIdx.x) * per, p.requests), r1 = min(r0 + per, p.requests);
    long long mine = 0;
    for (int r = r0; r < r1; ++r) mine += paged_request_units<TILE, UNIT>(p, paged_request(p, r));
    mine *= p.kv_heads;
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const long long x = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += x; }
    if (lane == 31) scratch[w] = upto;
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) { const long long x = scratch[i]; total += x; if (i < w) before += x; }
    upto += before;
    c.total = total;
    if (total == 0) return false;
    c.ctas = static_cast<int>(min(static_cast<long long>(gridDim.x), (total + min_units - 1) / min_units));
    if (static_cast<int>(blockIdx.x) >= c.ctas) return false;
    c.lo = total * blockIdx.x / c.ctas;
    c.hi = total * (blockIdx.x + 1) / c.ctas;
    __syncthreads();
    if (upto - mine <= c.lo && c.lo < upto) {
        long long at = upto - mine;
        int r = r0;
        for (;; ++r) {
            const long long n = paged_request_units<TILE, UNIT>(p, paged_request(p, r)) * p.kv_heads;
            if (c.lo < at + n) break;
            at += n;
        }
        scratch[0] = at; scratch[1] = r;
    }
    __syncthreads();
    long long at = scratch[0];
    c.r = static_cast<int>(scratch[1]);
    c.q = paged_request(p, c.r);
    for (c.t = 0;; ++c.t) {
        c.units = paged_tile_units<TILE, UNIT>(p, c.q, c.t);
        if (c.lo < at + static_cast<long long>(c.units) * p.kv_heads) break;
        at += static_cast<long long>(c.units) * p.kv_heads;
    }
    c.h = static_cast<int>((c.lo - at) / c.units);
    c.item = at + static_cast<long long>(c.h) * c.units;
    return true;
}
// To the next item; the caller has checked that there is one (c.item + c.units < c.total).
template <int TILE, int UNIT>
__device__ __forceinline__ void paged_next(const PagedParams& p, PagedCursor& c) {
    c.item += c.units;
    if (++c.h < p.kv_heads) return;
    c.h = 0;
    ++c.t;
    while (c.t * TILE >= c.q.rows) { c.t = 0; ++c.r; c.q = paged_request(p, c.r); }
    c.units = paged_tile_units<TILE, UNIT>(p, c.q, c.t);
}
// CTA whose stretch holds unit u.
__device__ __forceinline__ int paged_cta_of(const PagedCursor& c, long long u) { return static_cast<int>(((u + 1) * c.ctas - 1) / c.total); }

__device__ __forceinline__ float paged_clamp_scale(float s) { return fminf(fmaxf(s, 0x1p-40f), 0x1p72f); }

__device__ __forceinline__ void paged_store2(__nv_bfloat16* p, float a, float b) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b); }
__device__ __forceinline__ void paged_store2(__half* p, float a, float b) { *reinterpret_cast<__half2*>(p) = __floats2half2_rn(a, b); }

// Result of row `row` of the item from its sum `o` (values d, d + 1), weight `l` and reference maximum `m` (log2 units).
template <typename T, int D>
__device__ __forceinline__ void paged_finish2(const PagedParams& p, const PagedCursor& c, int row, int d, float o0, float o1, float m, float l) {
    const int token = row / p.group, head = c.h * p.group + (row - token * p.group);
    const size_t at = static_cast<size_t>(c.q.start) + token;
    const bool none = l == 0.0f;                                   // no key seen: zero and -inf
    const float inv = none ? 0.0f : 1.0f / l;
    paged_store2(static_cast<T*>(p.out) + at * p.out_stride + static_cast<size_t>(head) * D + d, none ? 0.0f : o0 * inv, none ? 0.0f : o1 * inv);
    if (p.lse && d == 0) p.lse[at * (static_cast<size_t>(p.group) * p.kv_heads) + head] = none ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

// A part of a split item has left its sums in this CTA's partial slot: announce it and, when all parts are there, join them.
// `rows` rows from tile row 0; scratch: at least (parts + 1) * rows * 2 floats of shared memory.  Called by all threads.
template <typename T, int D, int THREADS, int TILE>
__device__ __forceinline__ void paged_join(const PagedParams& p, const PagedCursor& c, int rows, int row0, float* scratch, int* flag) {
    const int first = paged_cta_of(c, c.item), last = paged_cta_of(c, c.item + c.units - 1);
    const int parts = last - first + 1;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        const int before = atomicAdd(p.counters + first, 1);
        *flag = before == parts - 1;
        if (before == parts - 1) p.counters[first] = 0;            // as the next call finds it
    }
    __syncthreads();
    if (!*flag) return;
    __threadfence();
    constexpr size_t SLOT = static_cast<size_t>(TILE) * (D + 2);
    auto slot = [&](int i) { return p.partials + (static_cast<size_t>(first + i) * 2 + (i == 0 ? 1 : 0)) * SLOT; };
    // factors of every part for every row: f[i][row] = 2^(m_i - m); the row's m and 1 / weight
    float* f = scratch;
    float* ml = scratch + static_cast<size_t>(parts) * rows;
    for (int i = threadIdx.x; i < parts * rows; i += THREADS) f[i] = __ldcg(slot(i / rows) + TILE * D + i % rows);
    __syncthreads();
    for (int row = threadIdx.x >> 5; row < rows; row += THREADS / 32) {      // one warp per row
        const int lane = threadIdx.x & 31;
        float m = -INFINITY;
        for (int i = lane; i < parts; i += 32) m = fmaxf(m, f[i * rows + row]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float ref = m == -INFINITY ? 0.0f : m;
        float l = 0.0f;
        for (int i = lane; i < parts; i += 32) {
            const float e = ex2_approx(f[i * rows + row] - ref);
            f[i * rows + row] = e;
            l += e * __ldcg(slot(i) + TILE * (D + 1) + row);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (lane == 0) { ml[2 * row] = ref; ml[2 * row + 1] = l; }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < rows * (D / 2); e += THREADS) {
        const int row = e / (D / 2), d = (e % (D / 2)) * 2;
        float o0 = 0.0f, o1 = 0.0f;
#pragma unroll 4
        for (int i = 0; i < parts; ++i) {
            const float2 v = __ldcg(reinterpret_cast<const float2*>(slot(i) + row * D + d));
            const float w = f[i * rows + row];
            o0 = fmaf(v.x, w, o0); o1 = fmaf(v.y, w, o1);
        }
        paged_finish2<T, D>(p, c, row0 + row, d, o0, o1, ml[2 * row], ml[2 * row + 1]);
    }
    __syncthreads();
}

}  // namespace b200
