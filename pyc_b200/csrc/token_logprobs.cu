// Log probabilities of given tokens, entropy and the top alternatives from rows of logits, and the gradient
// (formulas and meaning: include/pyc_b200.h).  PyC has no counterpart; the row softmax is in elementwise.cu.
//
// Forward: one pass over the row.  Each thread keeps a reference R >= log2(e) x of its elements, s = sum 2^y and t = sum y 2^y
// with y = log2(e) x - R, one fused multiply-add with a single rounding; joined, lse = (R + log2 s) ln 2 and entropy =
// (log2 s - t / s) ln 2.  Bound by reading the logits as long as an element takes fewer than nine issue slots: packed clamp and
// maximum on 16-bit pairs, packed f32 arithmetic, one exponential.
//
// The alternatives come out of the same pass.  The k-th largest of the THREADS threads' maxima, tau, is a lower bound of the k-th
// largest logit (k distinct elements reach it), and only threads whose maximum reaches tau can hold one.  The threads keep a
// maximum for each of up to 8 stretches of the row too, so that what is read again are some twenty eighths of a thread's
// elements, 4 % of the row (whole threads' shares were 30 %, for with 900 rows under way a row has left L2: 129 us instead of
// 119 us at 2048 x 131072 bf16); what reaches tau is ranked.  tau is found by one warp, by a
// bisection over the ordered bits.  Many ties at tau (coarse logits, a vocabulary masked down to a few tokens) end in a scan of the
// row from its start, which is where the ties that count are; see top_of_slice.
//
// Measured: 2048 x 131072 bf16 (537 MB) with 20 alternatives 119 us = 4.5 TB/s, bound by issue slots; 16 x 32768 f32 10.5 us.
//
// Rows are taken by one CTA each; where there are fewer rows than the SMs can hold, a cluster of 2, 4 or 8 CTAs shares a row
// and its first CTA joins the others' statistics and candidates through distributed shared memory.
//
// What lies at the lower end of the type's range (-inf, the lowest value that masks are made of) is clamped to FLOOR on the way
// in, so that nothing multiplies 0 by infinity; a row whose maximum is FLOOR (all masked) is done again exactly.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"
#include "math.cuh"

namespace b200 {
namespace {

constexpr int LT = 256;
constexpr int CTAS_PER_SM = 6;
constexpr int MAX_TOP = 32;
constexpr int MAX_CAND = 1024;
constexpr int SEGS = 8, MAX_EQ = 64, MAX_LIST = MAX_TOP * SEGS + MAX_EQ;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// Per type: 16-byte vectors of N elements as f32, clamped to the type's lowest value (NaN stays), with their maximum.
template <typename T> struct Logits;
template <> struct Logits<float> {
    static constexpr int N = 4, F32_BITS = 32;
    static __device__ __forceinline__ float lowest() { return -3.4028234663852886e38f; }
    static __device__ __forceinline__ float floor() { return -0x1.6p127f; }      // log2(e) times it is still finite
    static __device__ __forceinline__ float one(const float* p) { return *p; }
    static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
    static __device__ __forceinline__ float unpack(const uint4& u, float (&f)[4]) {
        f[0] = max_nan(__uint_as_float(u.x), floor()); f[1] = max_nan(__uint_as_float(u.y), floor());
        f[2] = max_nan(__uint_as_float(u.z), floor()); f[3] = max_nan(__uint_as_float(u.w), floor());
        return max_nan(max_nan(f[0], f[1]), max_nan(f[2], f[3]));
    }
    static __device__ __forceinline__ void raw(const uint4& u, float (&f)[4]) {
        f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[4]) { return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])); }
};
template <> struct Logits<__nv_bfloat16> {
    static constexpr int N = 8, F32_BITS = 16;
    static __device__ __forceinline__ float lowest() { return -3.3895313892515355e38f; }
    static __device__ __forceinline__ float floor() { return -0x1.6p127f; }
    static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) { uint32_t d; asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b)); return d; }
    static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
    static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
    static __device__ __forceinline__ float unpack(const uint4& u, float (&f)[8]) {
        constexpr uint32_t LOW = 0xff30ff30u;
        const uint32_t a = max2(u.x, LOW), b = max2(u.y, LOW), c = max2(u.z, LOW), d = max2(u.w, LOW), m = max2(max2(a, b), max2(c, d));
        f[0] = lo(a); f[1] = hi(a); f[2] = lo(b); f[3] = hi(b); f[4] = lo(c); f[5] = hi(c); f[6] = lo(d); f[7] = hi(d);
        return max_nan(lo(m), hi(m));
    }
    static __device__ __forceinline__ void raw(const uint4& u, float (&f)[8]) {
        f[0] = lo(u.x); f[1] = hi(u.x); f[2] = lo(u.y); f[3] = hi(u.y); f[4] = lo(u.z); f[5] = hi(u.z); f[6] = lo(u.w); f[7] = hi(u.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) { const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t*>(&h); }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <> struct Logits<__half> {
    static constexpr int N = 8, F32_BITS = 19;
    static __device__ __forceinline__ float lowest() { return -65504.0f; }
    static __device__ __forceinline__ float floor() { return -65504.0f; }
    static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
    static __device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) { uint32_t d; asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b)); return d; }
    static __device__ __forceinline__ float2 both(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ void split(uint32_t a, uint32_t b, uint32_t c, uint32_t d, float (&f)[8]) {
        const float2 p = both(a), q = both(b), r = both(c), s = both(d);
        f[0] = p.x; f[1] = p.y; f[2] = q.x; f[3] = q.y; f[4] = r.x; f[5] = r.y; f[6] = s.x; f[7] = s.y;
    }
    static __device__ __forceinline__ float unpack(const uint4& u, float (&f)[8]) {
        constexpr uint32_t LOW = 0xfbfffbffu;
        const uint32_t a = max2(u.x, LOW), b = max2(u.y, LOW), c = max2(u.z, LOW), d = max2(u.w, LOW);
        split(a, b, c, d, f);
        const float2 m = both(max2(max2(a, b), max2(c, d)));
        return max_nan(m.x, m.y);
    }
    static __device__ __forceinline__ void raw(const uint4& u, float (&f)[8]) { split(u.x, u.y, u.z, u.w, f); }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) { const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t*>(&h); }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

struct Stats { float r, s, t; };          // reference (in log2), sum 2^y, sum y 2^y
// The same sums about the reference r >= a.r.  What vanishes contributes nothing, however large its distance (0 * inf).
__device__ __forceinline__ Stats about(const Stats& a, float r) {
    const float d = a.r == r ? 0.0f : a.r - r, e = a.s * ex2_approx(d);
    return Stats{r, e, e > 0.0f ? fmaf(e, d, a.t * ex2_approx(d)) : 0.0f};
}
__device__ __forceinline__ Stats warp_join(const Stats& a) {
    float r = a.r;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, o));
    Stats c = about(a, r);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { c.s += __shfl_xor_sync(0xffffffffu, c.s, o); c.t += __shfl_xor_sync(0xffffffffu, c.t, o); }
    return c;
}

// Values ordered as unsigned numbers (minus zero with plus zero), and back.
__device__ __forceinline__ uint32_t ordered(float v) { const uint32_t u = __float_as_uint(v + 0.0f); return u & 0x80000000u ? ~u : u | 0x80000000u; }
__device__ __forceinline__ float from_ordered(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
// Larger value first, then the lower index: one number, never 0.
__device__ __forceinline__ unsigned long long key_of(float v, uint32_t index) { return (static_cast<unsigned long long>(ordered(v)) << 32) | (0xffffffffu - index); }

// The part of a row that a CTA reads: single elements up to the first 16-byte boundary (first CTA), vectors, single elements.
struct Slice { uint32_t head, tail, tail0, v0, v1, base, chunk; };      // vectors [v0, v1), vector v holds elements base + v * N ..; stretches of `chunk` vectors

struct Shared {
    Stats warp[LT / 32], all;
    unsigned long long cand[MAX_CAND];
    unsigned long long top[MAX_TOP];       // the slice's, sorted; 0: none
    uint32_t who[MAX_LIST], tmax[LT], seg[SEGS][LT];       // who: thread | stretch << 8
    uint32_t gt_threads, gt, eq, tau, other, scan[LT / 32];
    int bad;
};

// All elements of `lists` shares (share_of(i): thread | stretch << 8; a thread's single elements belong to its stretch 0), in
// no order: f(value, index).  Called by the whole CTA; the vectors are dealt out over its threads, four loads in flight each.
template <typename T, typename W, typename F>
__device__ __forceinline__ void read_shares(const T* x, const Slice& sl, uint32_t lists, const W& share_of, const F& f) {
    constexpr int N = Logits<T>::N, U = 4;
    const uint32_t per = sl.chunk / LT, all = lists * per;
    for (uint32_t i0 = threadIdx.x; i0 < all; i0 += U * LT) {
        uint4 u[U];
        uint32_t v[U];
#pragma unroll
        for (int y = 0; y < U; ++y) {
            const uint32_t i = i0 + y * LT;
            v[y] = sl.v1;
            if (i < all) {
                const uint32_t share = share_of(i / per);
                v[y] = sl.v0 + (share >> 8) * sl.chunk + (i % per) * LT + (share & 255u);
            }
            u[y] = v[y] < sl.v1 ? __ldg(reinterpret_cast<const uint4*>(x + sl.base) + v[y]) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int y = 0; y < U; ++y) {
            if (v[y] >= sl.v1) continue;
            float e[N];
            Logits<T>::raw(u[y], e);
#pragma unroll
            for (int j = 0; j < N; ++j) f(e[j], sl.base + v[y] * N + j);
        }
    }
    for (uint32_t i = threadIdx.x; i < lists; i += LT) {
        const uint32_t who = share_of(i);
        if (who < sl.head) f(Logits<T>::one(x + who), who);                 // stretch 0 only: the others' numbers are larger
        if (who < sl.tail) f(Logits<T>::one(x + sl.tail0 + who), sl.tail0 + who);
    }
}
// Element i of the slice in the order of the row.
__device__ __forceinline__ uint32_t slice_size(const Slice& sl, int n) { return sl.head + (sl.v1 - sl.v0) * n + sl.tail; }
__device__ __forceinline__ uint32_t slice_at(const Slice& sl, int n, uint32_t i) {
    if (i < sl.head) return i;
    i -= sl.head;
    const uint32_t mid = (sl.v1 - sl.v0) * n;
    return i < mid ? sl.base + sl.v0 * n + i : sl.tail0 + (i - mid);
}

// The slice's k largest by (value, lower index) into sh.top.  sh.seg: the threads' maxima of their clamped elements in each of
// `segs` stretches, ordered (0: none).
template <typename T>
__device__ void top_of_slice(const T* x, const Slice& sl, int k, int segs, Shared& sh) {
    constexpr int N = Logits<T>::N;
    const float low = Logits<T>::lowest();
    uint32_t mine = 0;
    for (int y = 0; y < segs; ++y) mine = max(mine, sh.seg[y][threadIdx.x]);
    if (threadIdx.x < MAX_TOP) sh.top[threadIdx.x] = 0;
    if (threadIdx.x == 0) { sh.gt_threads = 0; sh.gt = 0; sh.eq = 0; sh.other = 0; }
    sh.tmax[threadIdx.x] = mine;
    __syncthreads();
    if (threadIdx.x < 32) {
        // tau: the largest value that k threads' maxima reach; 0, below every value, when fewer than k threads have elements.  Only
        // the bits of f32 that the type fills; those below are all 0 (positive) or, ordered, all 1 (negative).
        constexpr int BITS = Logits<T>::F32_BITS;
        uint32_t v[LT / 32], tau = 0;
#pragma unroll
        for (int i = 0; i < LT / 32; ++i) v[i] = sh.tmax[i * 32 + threadIdx.x];
#pragma unroll 1
        for (int b = 31; b >= 32 - BITS; --b) {
            const uint32_t trial = tau | (1u << b);
            int c = 0;
#pragma unroll
            for (int i = 0; i < LT / 32; ++i) c += v[i] >= trial;
            if (__reduce_add_sync(0xffffffffu, c) >= k) tau = trial;
        }
        if (BITS < 32 && tau != 0 && !(tau & 0x80000000u)) tau |= static_cast<uint32_t>((1ull << (32 - BITS)) - 1);
        if (threadIdx.x == 0) sh.tau = tau;
    }
    __syncthreads();
    const uint32_t tau = sh.tau;
    const bool few = tau == 0;
    const float tau_v = from_ordered(tau);
    const bool masked = !few && tau_v <= Logits<T>::floor();      // what the clamp has made equal: told apart below
    if (mine != 0 && mine >= tau)
        for (int y = 0; y < segs; ++y) {
            const uint32_t m = sh.seg[y][threadIdx.x], share = threadIdx.x | (y << 8);
            if (m != 0 && m > tau) sh.who[atomicAdd(&sh.gt_threads, 1)] = share;              // fewer than k threads, SEGS each
            else if (m != 0 && m == tau) { const uint32_t e = atomicAdd(&sh.eq, 1); if (e < MAX_EQ) sh.who[MAX_LIST - 1 - e] = share; }
        }
    __syncthreads();
    const uint32_t gt_threads = sh.gt_threads, eq_threads = sh.eq;
    const bool scan = masked || eq_threads > MAX_EQ;
    // candidates above tau (few: all), and with few threads at tau those that equal it
    const uint32_t lists = gt_threads + (scan ? 0 : eq_threads);
    read_shares<T>(x, sl, lists, [&](uint32_t i) { return i < gt_threads ? sh.who[i] : sh.who[MAX_LIST - 1 - (i - gt_threads)]; }, [&](float v, uint32_t index) {
        if (few || (scan ? ordered(v) > tau : ordered(v) >= tau)) {
            const uint32_t at = atomicAdd(&sh.gt, 1);
            if (at < MAX_CAND) sh.cand[at] = key_of(v, index);
        }
    });
    __syncthreads();
    uint32_t n = sh.gt;
    if (n <= MAX_CAND && scan && n < static_cast<uint32_t>(k)) {
        // ties at tau: the lowest indices, in order.  masked: first the elements of the lowest value, then -inf; they are kept apart
        // in the two halves of what is left of the buffer (n < 32 is taken).  Anything else down there goes the slow way.
        const uint32_t need = k - n, size = slice_size(sl, N);
        uint32_t found = 0, found_inf = 0;
        for (uint32_t i0 = 0; i0 < size && (masked || found < need); i0 += LT) {
            const uint32_t i = i0 + threadIdx.x;
            const uint32_t index = i < size ? slice_at(sl, N, i) : 0;
            const float v = i < size ? Logits<T>::one(x + index) : INFINITY;
            const bool hit = i < size && (masked ? v == low : ordered(v) == tau), inf = masked && v == -INFINITY;
            if (masked && i < size && v <= Logits<T>::floor() && !hit && !inf) sh.other = 1;
            const unsigned mh = __ballot_sync(0xffffffffu, hit), mi = __ballot_sync(0xffffffffu, inf);
            const uint32_t w = threadIdx.x >> 5, lane = threadIdx.x & 31;
            if (lane == 0) sh.scan[w] = __popc(mh) | (__popc(mi) << 16);
            __syncthreads();
            uint32_t before = 0, total = 0;
#pragma unroll
            for (uint32_t y = 0; y < LT / 32; ++y) { total += sh.scan[y]; before += y < w ? sh.scan[y] : 0; }
            const uint32_t at = found + (before & 0xffffu) + __popc(mh & ((1u << lane) - 1u)), ai = found_inf + (before >> 16) + __popc(mi & ((1u << lane) - 1u));
            if (hit && at < need) sh.cand[n + at] = key_of(v, index);
            if (inf && ai < need) sh.cand[MAX_CAND / 2 + ai] = key_of(v, index);
            found += total & 0xffffu; found_inf += total >> 16;
            __syncthreads();
        }
        found = min(found, need);
        const uint32_t rest = min(found_inf, need - found);
        if (threadIdx.x < rest) sh.cand[n + found + threadIdx.x] = sh.cand[MAX_CAND / 2 + threadIdx.x];
        n += found + rest;
        __syncthreads();
    }
    if (n <= MAX_CAND && !sh.other) {
        // the rank of a candidate is the number of larger ones; keys are distinct
        for (uint32_t i = threadIdx.x; i < n; i += LT) {
            const unsigned long long mine_key = sh.cand[i];
            uint32_t rank = 0;
            for (uint32_t y = 0; y < n; ++y) rank += sh.cand[y] > mine_key;
            if (rank < static_cast<uint32_t>(k)) sh.top[rank] = mine_key;
        }
        __syncthreads();
        return;
    }
    // more than MAX_CAND elements above tau in the shares of fewer than k threads, or values between the lowest and FLOOR: one after the other
    const uint32_t size = slice_size(sl, N);
    unsigned long long last = ~0ull;
    for (int r = 0; r < k; ++r) {
        unsigned long long best = 0;
        for (uint32_t i = threadIdx.x; i < size; i += LT) {
            const uint32_t index = slice_at(sl, N, i);
            const unsigned long long key = key_of(Logits<T>::one(x + index), index);
            if (key < last && key > best) best = key;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) { const unsigned long long y = __shfl_xor_sync(0xffffffffu, best, o); best = y > best ? y : best; }
        if ((threadIdx.x & 31) == 0) sh.cand[threadIdx.x >> 5] = best;
        __syncthreads();
        for (int y = 0; y < LT / 32; ++y) best = sh.cand[y] > best ? sh.cand[y] : best;
        if (threadIdx.x == 0) sh.top[r] = best;
        last = best;
        __syncthreads();
    }
}

__device__ __forceinline__ uint32_t peer_address(const void* p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
    return r;
}
__device__ __forceinline__ float peer_float(uint32_t a) { float v; asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory"); return v; }
__device__ __forceinline__ unsigned long long peer_u64(uint32_t a) { unsigned long long v; asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory"); return v; }
__device__ __forceinline__ void cluster_barrier() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }

template <typename T>
__global__ void __launch_bounds__(LT, CTAS_PER_SM)
token_logprobs_kernel(pyc_b200_token_logprobs_args p, int ctas) {
    constexpr int N = Logits<T>::N, U = 4;
    __shared__ Shared sh;
    const float low = Logits<T>::floor();
    const size_t row = blockIdx.x / ctas;
    const uint32_t part = blockIdx.x % ctas;              // = the rank in the cluster
    const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
    const uint32_t vocab = static_cast<uint32_t>(p.vocab);
    Slice sl;
    {
        const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
        const uint32_t lead = min(off ? N - off : 0u, vocab), nv = (vocab - lead) / N;
        sl.base = lead;
        sl.v0 = static_cast<uint32_t>(static_cast<uint64_t>(nv) * part / ctas); sl.v1 = static_cast<uint32_t>(static_cast<uint64_t>(nv) * (part + 1) / ctas);
        sl.head = part == 0 ? lead : 0;
        sl.tail0 = lead + nv * N;
        sl.tail = part + 1 == static_cast<uint32_t>(ctas) ? vocab - sl.tail0 : 0;
        const uint32_t step = U * LT;                     // a stretch is a whole number of loop steps, and there are at most SEGS
        sl.chunk = max((sl.v1 - sl.v0 + SEGS * step - 1) / (SEGS * step), 1u) * step;
    }
    if (threadIdx.x == 0) sh.bad = 0;
    int tok = -1;                                         // the given token's logit, asked for before all others
    float x_tok = 0.0f;
    bool given = false;
    if (threadIdx.x == 0 && part == 0) {
        tok = __ldg(p.tokens + row);
        given = tok >= 0 && static_cast<uint32_t>(tok) < vocab;
        if (given) x_tok = Logits<T>::one(x + tok);
    }

    // ---- the pass
    float tmax = low;                                     // the thread's maximum
    Stats a = {low * LOG2E, 0.0f, 0.0f};
    bool bad = false;
    auto raise = [&](float m) { tmax = m; a = about(a, m * LOG2E); };
    auto take = [&](float v) {
        v = max_nan(v, low);
        bad |= !(v < INFINITY);
        if (v > tmax) raise(v);
        const float y = fmaf(v, LOG2E, -a.r), e = ex2_approx(y);
        a.s += e; a.t = fmaf(e, y, a.t);
    };
    if (threadIdx.x < sl.head) take(Logits<T>::one(x + threadIdx.x));
    if (threadIdx.x < sl.tail) take(Logits<T>::one(x + sl.tail0 + threadIdx.x));
    const uint4* xv = reinterpret_cast<const uint4*>(x + sl.base);
    const unsigned long long log2e2 = f32x2_splat(LOG2E);
    unsigned long long s2 = 0, t2 = 0;                    // packed sums beside a.s, a.t: (0, 0)
    int segs = 0;
    float smax = tmax;                                    // of the stretch; single elements belong to stretch 0
    uint32_t seg_end = sl.v0 + sl.chunk;
    const bool singles = threadIdx.x < sl.head || threadIdx.x < sl.tail;
    auto end_stretch = [&](bool any) { sh.seg[segs++][threadIdx.x] = any ? ordered(smax) : 0; smax = low; };
    for (uint32_t v0 = sl.v0; v0 < sl.v1; v0 += U * LT) { // the same steps for all threads
        const uint32_t v = v0 + threadIdx.x;
        if (v0 == seg_end) { end_stretch(true); seg_end += sl.chunk; }      // all threads have elements in a stretch that is not the last
        uint4 u[U];
#pragma unroll
        for (int i = 0; i < U; ++i) u[i] = v + i * LT < sl.v1 ? __ldg(xv + v + i * LT) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (v + i * LT >= sl.v1) break;
            float f[N];
            const float m = Logits<T>::unpack(u[i], f);
            bad |= !(m < INFINITY);
            smax = fmaxf(smax, m);
            if (m > tmax) {
                float x0, x1;
                f32x2_unpack(s2, x0, x1); a.s += x0 + x1;
                f32x2_unpack(t2, x0, x1); a.t += x0 + x1;
                s2 = t2 = 0;
                raise(m);
            }
            const unsigned long long minus = f32x2_splat(-a.r);
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const unsigned long long y = f32x2_fma(f32x2_pack(f[j], f[j + 1]), log2e2, minus);
                float y0, y1;
                f32x2_unpack(y, y0, y1);
                const unsigned long long e = f32x2_pack(ex2_approx(y0), ex2_approx(y1));
                s2 = f32x2_add(s2, e);
                t2 = f32x2_fma(e, y, t2);
            }
        }
    }
    {
        float x0, x1;
        f32x2_unpack(s2, x0, x1); a.s += x0 + x1;
        f32x2_unpack(t2, x0, x1); a.t += x0 + x1;
    }
    end_stretch(seg_end - sl.chunk + threadIdx.x < sl.v1 || (segs == 0 && singles));
    __syncthreads();                                      // sh.bad is zero
    if (bad) sh.bad = 1;
    const Stats w = warp_join(a);
    if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5] = w;
    __syncthreads();
    if (threadIdx.x < 32) {
        const Stats c = warp_join(threadIdx.x < LT / 32 ? sh.warp[threadIdx.x] : Stats{low * LOG2E, 0.0f, 0.0f});
        if (threadIdx.x == 0) sh.all = c;
    }
    const bool slice_bad = sh.bad != 0;
    if (p.top_k && !slice_bad) top_of_slice<T>(x, sl, p.top_k, segs, sh);
    __syncthreads();

    // ---- the row: the first CTA joins the others
    if (ctas > 1) {
        cluster_barrier();
        if (part == 0) {
            if (threadIdx.x < 32) {
                Stats c = {low * LOG2E, 0.0f, 0.0f};
                bool broken = false;
                if (threadIdx.x < static_cast<uint32_t>(ctas)) {
                    const uint32_t at = peer_address(&sh.all, threadIdx.x);
                    c = Stats{peer_float(at), peer_float(at + 4), peer_float(at + 8)};
                    broken = __float_as_int(peer_float(peer_address(&sh.bad, threadIdx.x))) != 0;
                }
                c = warp_join(c);
                broken = __any_sync(0xffffffffu, broken);
                if (threadIdx.x == 0) { sh.all = c; sh.bad = broken; }
            }
            if (p.top_k) {
                // up to 8 sorted lists of up to 32 keys: 256 candidates
                unsigned long long key = 0;
                const int r = threadIdx.x / MAX_TOP, i = threadIdx.x % MAX_TOP;
                if (r < ctas) key = r == 0 ? sh.top[i] : peer_u64(peer_address(&sh.top[i], r));
                __syncthreads();
                sh.cand[threadIdx.x] = key;
                __syncthreads();
                uint32_t rank = 0;
                for (int y = 0; y < ctas * MAX_TOP; ++y) rank += sh.cand[y] > key;
                if (key && rank < static_cast<uint32_t>(p.top_k)) sh.top[rank] = key;
            }
        }
        cluster_barrier();                                // nobody leaves while its memory is read
        if (part != 0) return;
        __syncthreads();
    }
    const bool broken = sh.bad != 0;
    // natural logarithms from here on: of the sum, about the reference m
    float m = 0.0f, ln_s = 0.0f, mean = 0.0f;             // mean = sum p (x - m)
    const Stats all = sh.all;
    const bool redo = !broken && (all.r <= low * LOG2E || all.r > 1e30f);
    if (redo) {
        // nothing but masked logits, or ones beside which the clamp would show: the row once more, exactly, about its largest
        float big = -INFINITY;
        for (uint32_t i = threadIdx.x; i < vocab; i += LT) big = fmaxf(big, Logits<T>::one(x + i));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
        __syncthreads();
        if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5].r = big;
        __syncthreads();
        for (int i = 0; i < LT / 32; ++i) big = fmaxf(big, sh.warp[i].r);
        Stats c = {0.0f, 0.0f, 0.0f};
        for (uint32_t i = threadIdx.x; i < vocab; i += LT) {
            const float d = Logits<T>::one(x + i) - big, e = ex2_approx(d * LOG2E);
            if (e > 0.0f) { c.s += e; c.t = fmaf(e, d, c.t); }                   // not for -inf - (-inf)
        }
        c = warp_join(c);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5] = c;
        __syncthreads();
        c = sh.warp[0];
        for (int i = 1; i < LT / 32; ++i) { c.s += sh.warp[i].s; c.t += sh.warp[i].t; }
        m = big; ln_s = logf(c.s); mean = c.t / c.s;
    } else {
        ln_s = log2f(all.s); mean = all.t / all.s;        // in log2 units, taken back below
    }
    const bool none = redo && m == -INFINITY;
    const float nan = __int_as_float(0x7fffffff);
    constexpr float LN2 = 0.69314718055994531f;
    // a log probability is (x - m) - ln s: x - lse would lose ln s beside a large maximum
    auto log_p = [&](float v) { return broken ? nan : none ? -INFINITY : redo ? (v - m) - ln_s : v < low ? v - (all.r + ln_s) * LN2 : (fmaf(v, LOG2E, -all.r) - ln_s) * LN2; };
    if (threadIdx.x == 0) {
        p.logprob[row] = broken || given ? log_p(x_tok) : 0.0f;
        if (p.lse) p.lse[row] = broken ? nan : none ? -INFINITY : redo ? m + ln_s : (all.r + ln_s) * LN2;
        if (p.entropy) p.entropy[row] = broken ? nan : none ? 0.0f : fmaxf((ln_s - mean) * (redo ? 1.0f : LN2), 0.0f);
    }
    if (static_cast<int>(threadIdx.x) < p.top_k) {
        const unsigned long long key = sh.top[threadIdx.x];
        p.top_ids[row * p.top_k + threadIdx.x] = broken ? -1 : static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
        p.top_logprobs[row * p.top_k + threadIdx.x] = log_p(from_ordered(static_cast<uint32_t>(key >> 32)));
    }
}

// ---- gradient: reads and writes each element once, bound by that: 2048 x 131072 bf16 (1.07 GB) 159 us = 6.8 TB/s, 61 x 50001 f32 4.5 us.  One CTA per row and chunk of GRAD_CHUNK vectors; 16-byte
// accesses where logits and gradient lie equally to a 16-byte boundary, single elements otherwise.
constexpr int GRAD_U = 4, GRAD_CHUNK = LT * GRAD_U * 2;

template <typename T>
__global__ void __launch_bounds__(LT)
token_logprobs_grad_kernel(pyc_b200_token_logprobs_grad_args p, uint32_t chunks) {
    constexpr int N = Logits<T>::N;
    const size_t row = blockIdx.x / chunks;
    const uint32_t chunk = blockIdx.x % chunks, vocab = static_cast<uint32_t>(p.vocab);
    const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
    T* d = static_cast<T*>(p.grad_logits) + row * p.grad_stride;
    const float lse = __ldg(p.lse + row);
    const float u = p.grad_logprob ? __ldg(p.grad_logprob + row) : 0.0f, w = p.grad_entropy ? __ldg(p.grad_entropy + row) : 0.0f;
    const int tok = __ldg(p.tokens + row);
    const bool given = tok >= 0 && static_cast<uint32_t>(tok) < vocab;
    const float c = (given ? u : 0.0f) + (w != 0.0f ? w * __ldg(p.entropy + row) : 0.0f);
    const bool none = lse == -INFINITY;
    // -inf logits: log p is held at -1e30, so that p (c + w log p) is 0, not 0 * inf
    auto grad = [&](float v) {
        const float lp = max_nan(v - lse, -1e30f);
        return none ? 0.0f : -ex2_approx(lp * LOG2E) * fmaf(w, lp, c);
    };
    auto one = [&](uint32_t i) {
        float g = grad(Logits<T>::one(x + i));
        if (given && !none && i == static_cast<uint32_t>(tok)) g += u;
        Logits<T>::store(d + i, g);
    };
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T)), off_d = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(d) % 16 / sizeof(T));
    if (off != off_d) {
        const uint32_t i0 = chunk * (GRAD_CHUNK * N), i1 = min(vocab, i0 + GRAD_CHUNK * N);
        for (uint32_t i = i0 + threadIdx.x; i < i1; i += LT) one(i);
        return;
    }
    const uint32_t lead = min(off ? N - off : 0u, vocab), nv = (vocab - lead) / N, tail0 = lead + nv * N;
    if (chunk == 0) {
        if (threadIdx.x < lead) one(threadIdx.x);
        if (tail0 + threadIdx.x < vocab && threadIdx.x < N) one(tail0 + threadIdx.x);
    }
    const uint4* xv = reinterpret_cast<const uint4*>(x + lead);
    uint4* dv = reinterpret_cast<uint4*>(d + lead);
    const uint32_t end = min(nv, (chunk + 1) * GRAD_CHUNK);
    for (uint32_t v = chunk * GRAD_CHUNK + threadIdx.x; v < end; v += GRAD_U * LT) {
        uint4 r[GRAD_U];
#pragma unroll
        for (int i = 0; i < GRAD_U; ++i) if (v + i * LT < end) r[i] = xv[v + i * LT];
#pragma unroll
        for (int i = 0; i < GRAD_U; ++i) {
            if (v + i * LT >= end) break;
            float f[N];
            Logits<T>::raw(r[i], f);
#pragma unroll
            for (int y = 0; y < N; ++y) f[y] = grad(f[y]);
            const uint32_t at = lead + (v + i * LT) * N;
            if (given && !none && static_cast<uint32_t>(tok) - at < static_cast<uint32_t>(N)) {
#pragma unroll
                for (int y = 0; y < N; ++y) if (static_cast<uint32_t>(tok) == at + y) f[y] += u;
            }
            dv[v + i * LT] = Logits<T>::pack(f);
        }
    }
}

bool logits_ok(pyc_dtype t, size_t rows, size_t vocab, size_t stride) {
    if (t != PYC_DTYPE_F32 && t != PYC_DTYPE_BF16 && t != PYC_DTYPE_F16) { set_error("token logprobs: unsupported dtype %d", static_cast<int>(t)); return false; }
    if (rows == 0 || vocab == 0 || rows > 0x7fffffffull || vocab > 0x7fffffffull) { set_error("token logprobs: rows and vocab must be 1 .. 2^31 - 1"); return false; }
    if (stride < vocab) { set_error("token logprobs: row stride %zu below vocab %zu", stride, vocab); return false; }
    return true;
}
bool aligned_to(const void* q, pyc_dtype t) { return reinterpret_cast<uintptr_t>(q) % dtype_size(t) == 0; }

template <typename T>
int launch_scores(const pyc_b200_token_logprobs_args& p, cudaStream_t s) {
    // CTAs per row: the number that minimises waves x (bytes of a slice + FIXED + CLUSTER per CTA of the cluster), what a CTA's
    // beginning, alternatives and end take, and what a cluster adds, both in bytes of a CTA's share of the bandwidth (7 GB/s).
    // Measured with 1, 2, 4, 8: 16 rows of 32768 f32 13.0, 11.6, 10.5, 12.5 us; 2048 rows of 131072 bf16 119, 147, 202, 353 us.
    constexpr size_t FIXED = 72 * 1024, CLUSTER = 8 * 1024;
    const size_t slots = static_cast<size_t>(sm_count()) * CTAS_PER_SM, bytes = p.vocab * sizeof(T);
    int ctas = 1;
    size_t best = ~static_cast<size_t>(0);
    for (int c = 1; c <= 8; c *= 2) {
        const size_t cost = ((p.rows * c + slots - 1) / slots) * (bytes / c + FIXED + (c > 1 ? c * CLUSTER : 0));
        if (cost < best) { best = cost; ctas = c; }
    }
    if (p.rows * ctas > 0x7fffffffull) ctas = 1;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ctas; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(p.rows * ctas)); cfg.blockDim = dim3(LT); cfg.stream = s; cfg.attrs = &attr; cfg.numAttrs = ctas > 1 ? 1 : 0;
    B200_CUDA_OK(cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T>, p, ctas));
    count_launch();
    return 0;
}

template <typename T>
int launch_grad(const pyc_b200_token_logprobs_grad_args& p, cudaStream_t s) {
    const size_t chunks = (p.vocab + static_cast<size_t>(GRAD_CHUNK) * Logits<T>::N - 1) / (static_cast<size_t>(GRAD_CHUNK) * Logits<T>::N);
    if (p.rows * chunks > 0x7fffffffull) { set_error("token logprobs backward: rows * vocab is too large for one launch"); return -1; }
    token_logprobs_grad_kernel<T><<<static_cast<unsigned>(p.rows * chunks), LT, 0, s>>>(p, static_cast<uint32_t>(chunks));
    B200_CUDA_OK(cudaGetLastError());
    count_launch();
    return 0;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

int pyc_b200_token_logprobs(const pyc_b200_token_logprobs_args* a, void* stream) {
    if (!a || !a->logits || !a->tokens || !a->logprob) { set_error("token logprobs: NULL argument"); return -1; }
    pyc_b200_token_logprobs_args p = *a;
    if (!p.row_stride) p.row_stride = p.vocab;
    if (!logits_ok(p.dtype, p.rows, p.vocab, p.row_stride)) return -1;
    if (!aligned_to(p.logits, p.dtype)) { set_error("token logprobs: logits are not aligned to their type"); return -1; }
    if (p.top_k < 0 || p.top_k > MAX_TOP || static_cast<size_t>(p.top_k) > p.vocab) { set_error("token logprobs: top_k %d is not in 0 .. min(%d, vocab)", p.top_k, MAX_TOP); return -1; }
    if (p.top_k && (!p.top_ids || !p.top_logprobs)) { set_error("token logprobs: top_k without top_ids and top_logprobs"); return -1; }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (p.dtype == PYC_DTYPE_F32) return launch_scores<float>(p, s);
    if (p.dtype == PYC_DTYPE_BF16) return launch_scores<__nv_bfloat16>(p, s);
    return launch_scores<__half>(p, s);
}

int pyc_b200_token_logprobs_backward(const pyc_b200_token_logprobs_grad_args* a, void* stream) {
    if (!a || !a->logits || !a->tokens || !a->lse || !a->grad_logits) { set_error("token logprobs backward: NULL argument"); return -1; }
    if (a->grad_entropy && !a->entropy) { set_error("token logprobs backward: grad_entropy without entropy"); return -1; }
    pyc_b200_token_logprobs_grad_args p = *a;
    if (!p.row_stride) p.row_stride = p.vocab;
    if (!p.grad_stride) p.grad_stride = p.vocab;
    if (!logits_ok(p.dtype, p.rows, p.vocab, p.row_stride) || !logits_ok(p.dtype, p.rows, p.vocab, p.grad_stride)) return -1;
    if (!aligned_to(p.logits, p.dtype) || !aligned_to(p.grad_logits, p.dtype)) { set_error("token logprobs backward: logits or gradient are not aligned to their type"); return -1; }
    if (p.grad_logits == p.logits && p.grad_stride != p.row_stride) { set_error("token logprobs backward: in place needs equal strides"); return -1; }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (p.dtype == PYC_DTYPE_F32) return launch_grad<float>(p, s);
    if (p.dtype == PYC_DTYPE_BF16) return launch_grad<__nv_bfloat16>(p, s);
    return launch_grad<__half>(p, s);
}

}  // extern "C"
