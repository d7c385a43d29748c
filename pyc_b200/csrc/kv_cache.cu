// The 8-bit paged key/value cache: block tables and slot maps of a step (kv_plan), the return of finished requests'
// blocks (kv_release), and the quantising write of new keys and values (kv_write).  Layout and meaning of every array:
// include/pyc_b200.h.  PyC has no counterpart.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "internal.h"
#include "kv_cache.cuh"

namespace b200 {

namespace {

// ------------------------------------------------------------------------------------------------------------- plan --
// Two exclusive prefix sums over the requests (new tokens, new blocks), then one entry per new block and per new token.
// There is next to nothing to read or write (16 bytes per token), so what counts is latency: ONE launch.  Every CTA of a
// cluster repeats the scan over all requests in its own shared memory (8 bytes per request out of L2) and then fills its
// share of the entries, finding the request of an entry by binary search in the scanned array.  The cluster barrier in the
// middle lets the free count be updated in place: no CTA reads it after the barrier, CTA 0 writes it behind.
// Measured: 8 requests of one token 3.6 us, 2000 requests with 58 K new tokens 11 us (1 MB of tables; latency).
constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_MAX_REQUESTS = 16384;    // two int arrays in shared memory: 128 KB

__device__ __forceinline__ void plan_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Exclusive block scan of a pair of 64-bit sums; `total` gets the sums over the block.
__device__ __forceinline__ void block_scan2(long long& a, long long& b, long long (*warp_sums)[2], long long (&total)[2]) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const long long a0 = a, b0 = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) { a += x; b += y; }
    }
    if (lane == 31) { warp_sums[w][0] = a; warp_sums[w][1] = b; }
    __syncthreads();
    if (w == 0) {
        const bool in = lane < static_cast<int>(blockDim.x >> 5);
        long long x = in ? warp_sums[lane][0] : 0, y = in ? warp_sums[lane][1] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) { x += u; y += v; }
        }
        warp_sums[lane][0] = x; warp_sums[lane][1] = y;      // inclusive; the entries past the last warp repeat the total
    }
    __syncthreads();
    total[0] = warp_sums[31][0]; total[1] = warp_sums[31][1];
    a += (w ? warp_sums[w - 1][0] : 0) - a0;
    b += (w ? warp_sums[w - 1][1] : 0) - b0;
}

// Largest r with first[r] <= i, for i in [0, total): the request that entry i belongs to.  Requests without entries repeat
// the next one's start and are stepped over.
__device__ __forceinline__ int owner_of(const int* first, int n, int i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= i) lo = mid; else hi = mid;
    }
    return lo;
}

// The same for N times 32 entries of a warp, each time 32 in order; entries below 0 get request 0.  One search by all lanes together
// (lane x for the first of the x-th 32, lane N + x for the last) bounds the others to the requests between, which lie in
// different banks: 58 K tokens took 13.3 us with a whole search for each, for its bank conflicts, and take 11.3 us so.
template <int N>
__device__ __forceinline__ void owners_of(const int* first, int n, const int (&i)[N], int (&r)[N]) {
    const int lane = threadIdx.x & 31;
    int end = 0;
#pragma unroll
    for (int x = 0; x < N; ++x) {
        const int a = __shfl_sync(0xffffffffu, i[x], 0), b = __shfl_sync(0xffffffffu, i[x], 31);
        if (lane % (2 * N) == x) end = a;
        if (lane % (2 * N) == N + x) end = b;
    }
    const int bound = owner_of(first, n, end);
#pragma unroll
    for (int x = 0; x < N; ++x) {
        r[x] = __shfl_sync(0xffffffffu, bound, x);
        const int last = __shfl_sync(0xffffffffu, bound, N + x);
        for (int step = last > r[x] ? 1 << (31 - __clz(last - r[x])) : 0; step > 0; step >>= 1) {
            const int y = r[x] + step;
            if (y <= last && first[y] <= i[x]) r[x] = y;
        }
    }
}

__global__ void __launch_bounds__(PLAN_THREADS)
kv_plan_kernel(pyc_b200_kv_plan_args p, int block_shift) {
    extern __shared__ int plan_smem[];
    int* tok0 = plan_smem;                       // first new token of each request
    int* blk0 = plan_smem + p.requests;          // first new block
    __shared__ long long warp_sums[32][2];
    const int R = p.requests, bs = p.block_size;
    const int ctas = gridDim.x;                  // the grid is one cluster
    const int me = blockIdx.x * PLAN_THREADS + threadIdx.x, all = ctas * PLAN_THREADS;

    const long long free_count = min(max(static_cast<long long>(*p.free_count), 0ll), static_cast<long long>(p.num_blocks));
    const int per = (R + PLAN_THREADS - 1) / PLAN_THREADS;
    const int r0 = min(static_cast<int>(threadIdx.x) * per, R), r1 = min(r0 + per, R);
    long long toks = 0, blks = 0;
    int bad = 0;
    for (int r = r0; r < r1; ++r) {
        const long long c = p.context_lens[r], n = p.new_lens[r];
        if (c < 0 || n < 0) { bad |= 1; continue; }
        if (c + n > static_cast<long long>(p.max_blocks) * bs) { bad |= 2; continue; }
        toks += n;
        blks += ((c + n + bs - 1) >> block_shift) - ((c + bs - 1) >> block_shift);
    }
    long long t_at = toks, b_at = blks, total[2];
    block_scan2(t_at, b_at, warp_sums, total);
    bad |= (total[0] > p.max_tokens ? 4 : 0) | (total[1] > free_count ? 8 : 0);
    bad = __syncthreads_or(bad & 1) ? (bad | 1) : bad;
    bad = __syncthreads_or(bad & 2) ? (bad | 2) : bad;

    if (bad) {
        for (int i = me; i <= R; i += all) {
            p.query_start[i] = 0;
            if (i < R) p.seq_lens[i] = p.context_lens[i];
        }
        for (int t = me; t < p.max_tokens; t += all) { p.slot_map[t] = -1; p.positions[t] = 0; p.token_request[t] = -1; }
        plan_cluster_sync();
        if (me == 0) {
            p.result[0] = bad; p.result[1] = 0; p.result[2] = 0;
            p.result[3] = (bad & 8) ? static_cast<int>(min(total[1] - free_count, static_cast<long long>(INT_MAX))) : 0;
            if (p.free_count_out) *p.free_count_out = *p.free_count;
        }
        return;
    }

    for (int r = r0; r < r1; ++r) {
        const int c = p.context_lens[r], n = p.new_lens[r];
        tok0[r] = static_cast<int>(t_at); blk0[r] = static_cast<int>(b_at);
        if (blockIdx.x == 0) { p.query_start[r] = static_cast<int>(t_at); p.seq_lens[r] = c + n; }
        t_at += n;
        b_at += ((c + n + bs - 1) >> block_shift) - ((c + bs - 1) >> block_shift);
    }
    const int T = static_cast<int>(total[0]), B = static_cast<int>(total[1]);
    if (me == 0) { p.query_start[R] = T; p.result[0] = 0; p.result[1] = T; p.result[2] = B; p.result[3] = 0; }
    __syncthreads();
    plan_cluster_sync();                         // result[0] is set before any CTA adds a flag to it; free_count has been read by all
    if (me == 0) *(p.free_count_out ? p.free_count_out : p.free_count) = static_cast<int>(free_count) - B;

    const int* top = p.free_blocks + (free_count - 1);
    bool outside = false;
    for (int i = me; i < B; i += all) {
        const int r = owner_of(blk0, R, i);
        const int have = (p.context_lens[r] + bs - 1) >> block_shift;
        const int id = top[-i];
        p.block_table[static_cast<size_t>(r) * p.max_blocks + have + (i - blk0[r])] = id;
        outside |= static_cast<unsigned>(id) >= static_cast<unsigned>(p.num_blocks);
    }
    // 2000 requests, 58 K tokens: 11.3 us with four tokens at once, 13.9 with one; 8 tokens: 4.2 and 3.6.  So four where there is a cluster.
    auto fill = [&](auto n) {
        constexpr int AT_ONCE = decltype(n)::value;          // tokens per thread and step: their searches and loads overlap
        for (long long t0 = me; t0 - (threadIdx.x & 31) < p.max_tokens; t0 += static_cast<long long>(AT_ONCE) * all) {
            int at[AT_ONCE], r[AT_ONCE], pos[AT_ONCE], id[AT_ONCE];
#pragma unroll
            for (int x = 0; x < AT_ONCE; ++x) at[x] = static_cast<int>(min(t0 + static_cast<long long>(x) * all, static_cast<long long>(T) - 1));
            if constexpr (AT_ONCE == 1) r[0] = owner_of(tok0, R, max(at[0], 0));
            else owners_of<AT_ONCE>(tok0, R, at, r);
#pragma unroll
            for (int x = 0; x < AT_ONCE; ++x) {
                const int c = T > 0 ? p.context_lens[r[x]] : 0;
                pos[x] = c + (at[x] - tok0[r[x]]);
                const int have = (c + bs - 1) >> block_shift, j = pos[x] >> block_shift;
                // a block of this step comes straight from the free list: its table entry may be written by another CTA meanwhile
                const int* from = j < have ? p.block_table + static_cast<size_t>(r[x]) * p.max_blocks + j : top - (blk0[r[x]] + j - have);
                id[x] = T > 0 ? *from : 0;
            }
#pragma unroll
            for (int x = 0; x < AT_ONCE; ++x) {
                const long long t = t0 + static_cast<long long>(x) * all;
                if (t >= p.max_tokens) break;
                const bool some = t < T, in = some && static_cast<unsigned>(id[x]) < static_cast<unsigned>(p.num_blocks);
                outside |= some && !in;
                p.slot_map[t] = in ? static_cast<long long>(id[x]) * bs + (pos[x] & (bs - 1)) : -1ll;
                p.positions[t] = some ? pos[x] : 0;
                p.token_request[t] = some ? r[x] : -1;
            }
        }
    };
    if (ctas == 1) fill(std::integral_constant<int, 1>{});
    else fill(std::integral_constant<int, 4>{});
    if (outside) atomicOr(p.result, 16);
}

// Blocks of finished requests, pushed behind the free list in the order of the requests.  One CTA: a scan of the block
// counts, then one table entry per thread and step.
__global__ void __launch_bounds__(PLAN_THREADS)
kv_release_kernel(int R, int bs, int block_shift, int num_blocks, int max_blocks, const int* __restrict__ finished, int* __restrict__ context_lens,
                  int* __restrict__ table, int* __restrict__ free_blocks, int* __restrict__ free_count) {
    extern __shared__ int plan_smem[];
    int* blk0 = plan_smem;
    __shared__ long long warp_sums[32][2];
    const long long count = min(max(static_cast<long long>(*free_count), 0ll), static_cast<long long>(num_blocks));
    const int per = (R + PLAN_THREADS - 1) / PLAN_THREADS;
    const int r0 = min(static_cast<int>(threadIdx.x) * per, R), r1 = min(r0 + per, R);
    auto held = [&](int r) -> int {
        if (finished[r] == 0) return 0;
        const long long c = min(max(static_cast<long long>(context_lens[r]), 0ll), static_cast<long long>(max_blocks) * bs);
        return static_cast<int>((c + bs - 1) >> block_shift);
    };
    long long n = 0, zero = 0, total[2];
    for (int r = r0; r < r1; ++r) n += held(r);
    long long at = n;
    block_scan2(at, zero, warp_sums, total);
    for (int r = r0; r < r1; ++r) { blk0[r] = static_cast<int>(min(at, static_cast<long long>(INT_MAX))); at += held(r); }
    __syncthreads();
    // a list that would outgrow the pool means that a block was handed in twice: what does not fit is dropped
    const int B = static_cast<int>(min(total[0], num_blocks - count));
    for (int i = threadIdx.x; i < B; i += PLAN_THREADS) {
        const int r = owner_of(blk0, R, i);
        int* entry = table + static_cast<size_t>(r) * max_blocks + (i - blk0[r]);
        free_blocks[count + i] = *entry;
        *entry = -1;
    }
    __syncthreads();
    for (int r = r0; r < r1; ++r)
        if (finished[r] != 0) context_lens[r] = 0;
    if (threadIdx.x == 0) *free_count = static_cast<int>(count) + B;
}

// ------------------------------------------------------------------------------------------------------------ write --
// Bound by reading the 16-bit values and writing the codes, or by latency for single tokens.  One CTA per (group of tokens, head,
// keys | values) takes the runs that begin in its group one after the other.  A thread holds eight 16-byte vectors, a CTA
// block_size * head_dim / 2048 warps, so that a whole block's values of a head are loaded at once, kept in registers while
// their largest magnitude is found, and written as codes: every value is read once.
// Measured: 64 single tokens (8 heads of 128) 2.9 us; 13 K tokens of prompts (82 MB) 19 us = 4.3 TB/s; reading the values twice, once
// for the magnitude, took 100 us.
template <typename T> struct KvIn;
template <> struct KvIn<__nv_bfloat16> {
    static constexpr uint32_t INF = 0x7f80;
    static __device__ __forceinline__ float widen(uint32_t bits) { return __uint_as_float(bits << 16); }
    static __device__ __forceinline__ void unpack(uint32_t w, float& a, float& b) { a = __uint_as_float(w << 16); b = __uint_as_float(w & 0xffff0000u); }
};
template <> struct KvIn<__half> {
    static constexpr uint32_t INF = 0x7c00;
    static __device__ __forceinline__ float widen(uint32_t bits) { return __half2float(__ushort_as_half(static_cast<unsigned short>(bits))); }
    static __device__ __forceinline__ void unpack(uint32_t w, float& a, float& b) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w)); a = f.x; b = f.y;
    }
};

struct KvWriteParams {
    const void* x[2];
    size_t stride[2];
    uint8_t* cache[2];
    float* scale[2];
    const long long* slots;
    int tokens, heads, bs, shift, num_blocks, group;
};

// Largest magnitude of a thread's values as 16-bit bits (magnitudes order as their bits); FINITE: infinities and NaN left out.
template <bool FINITE, int VECS>
__device__ __forceinline__ uint32_t max_bits(const uint4 (&u)[VECS], uint32_t inf) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t a = w[j] & 0x7fff7fffu;
            if (FINITE) a = ((a & 0xffffu) < inf ? a & 0xffffu : 0u) | ((a >> 16) < inf ? a & 0xffff0000u : 0u);
            m = __vmaxu2(m, a);
        }
    }
    return max(m & 0xffffu, m >> 16);
}

__device__ __forceinline__ uint32_t kv_pack4(float a, float b, float c, float d) {
    const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}

// W: warps per CTA.
template <typename T, int D, int W>
__global__ void __launch_bounds__(W * 32, 32 / W)
kv_write_kernel(const __grid_constant__ KvWriteParams p) {
    constexpr int THREADS = W * 32, VECS = 8, PER_ROW = D / 8;               // vectors per row of a head
    const int lane = threadIdx.x & 31;
    const int head = blockIdx.y, which = blockIdx.z;
    const T* x = static_cast<const T*>(which ? p.x[1] : p.x[0]) + head * D;
    const size_t stride = which ? p.stride[1] : p.stride[0];
    float* scales = which ? p.scale[1] : p.scale[0];
    uint8_t* cache = which ? p.cache[1] : p.cache[0];
    const long long pool = static_cast<long long>(p.num_blocks) << p.shift;
    const int first = static_cast<int>(blockIdx.x) * p.group, last = min(first + p.group, p.tokens);
    for (int base = first; base < last; base += 32) {
        // tokens of these 32 that begin a run (the same in every warp)
        const int ti = base + lane;
        long long si = -1;
        bool leads = false;
        if (ti < last) {
            si = __ldg(p.slots + ti);
            if (si >= 0 && si < pool) leads = (si & (p.bs - 1)) == 0 || ti == 0 || __ldg(p.slots + ti - 1) != si - 1;
        }
        for (unsigned m = __ballot_sync(0xffffffffu, leads); m; m &= m - 1) {
            const int at = __ffs(m) - 1, t0 = base + at;
            const long long slot = __shfl_sync(0xffffffffu, si, at), block = slot >> p.shift;
            const int off = static_cast<int>(slot & (p.bs - 1));
            float* sp = scales + block * p.heads + head;
            const float old = *sp;
            // the run's tokens: consecutive slots up to the block's end.  A block has one run: where its last slot is the last token's, all are.
            const int most = min(p.bs - off, p.tokens - t0);
            int n = most;
            if (most > 1 && __ldg(p.slots + t0 + most - 1) != slot + most - 1) {
                n = 1;
                while (true) {
                    const int i = n + lane;
                    const bool more = i < most && __ldg(p.slots + t0 + i) == slot + i;
                    const unsigned run = __ballot_sync(0xffffffffu, more);
                    if (run == 0xffffffffu) { n += 32; continue; }
                    n += __ffs(~run) - 1;
                    break;
                }
            }
            uint4 u[VECS];
#pragma unroll
            for (int i = 0; i < VECS; ++i) {
                const int q = i * THREADS + threadIdx.x, r = q / PER_ROW;
                u[i] = r < n ? __ldg(reinterpret_cast<const uint4*>(x + static_cast<size_t>(t0 + r) * stride) + q % PER_ROW) : make_uint4(0, 0, 0, 0);
            }
            auto all = [&](uint32_t m) {                                     // the CTA's largest; also: everybody has read the old scale
                m = __reduce_max_sync(0xffffffffu, m);
                if constexpr (W > 1) {
                    __shared__ uint32_t warp_max[W];
                    if (lane == 0) warp_max[threadIdx.x >> 5] = m;
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < W; ++i) m = max(m, warp_max[i]);
                    __syncthreads();
                }
                return m;
            };
            uint32_t bits = all(max_bits<false>(u, KvIn<T>::INF));
            if (bits >= KvIn<T>::INF) bits = all(max_bits<true>(u, KvIn<T>::INF));
            int e = kv_scale_exponent(KvIn<T>::widen(bits));
            uint8_t* tile = cache + (static_cast<size_t>(block) * p.heads + head) * (static_cast<size_t>(p.bs) * D);
            if (off != 0) {
                e = max(e, kv_exponent_of_scale(old));
                const float again = old * exp2_int(-e);                      // old scale / new scale
                if (again != 1.0f) {
                    // codes that the block keeps, rounded again to the grown scale: 16 codes per thread and step
                    for (int i = threadIdx.x; i < off * D / 16; i += THREADS) {
                        uint4 v = reinterpret_cast<uint4*>(tile)[i];
                        uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 a = e4m3x2_to_float2(w[j] & 0xffffu), b = e4m3x2_to_float2(w[j] >> 16);
                            w[j] = kv_pack4(a.x * again, a.y * again, b.x * again, b.y * again);
                        }
                        reinterpret_cast<uint4*>(tile)[i] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            const float inv = exp2_int(-e);                                  // exact: the scale is a power of two
            uint2* dst = reinterpret_cast<uint2*>(tile + off * D);
#pragma unroll
            for (int i = 0; i < VECS; ++i) {
                const int q = i * THREADS + threadIdx.x;
                if (q / PER_ROW < n) {
                    const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
                    float f[8];
#pragma unroll
                    for (int j = 0; j < 4; ++j) { KvIn<T>::unpack(w[j], f[2 * j], f[2 * j + 1]); f[2 * j] *= inv; f[2 * j + 1] *= inv; }
                    dst[q] = make_uint2(kv_pack4(f[0], f[1], f[2], f[3]), kv_pack4(f[4], f[5], f[6], f[7]));
                }
            }
            if (threadIdx.x == 0) *sp = exp2_int(e);
        }
    }
}

template <typename T, int D>
int launch_kv_write(const KvWriteParams& p, cudaStream_t s) {
    const dim3 grid((p.tokens + p.group - 1) / p.group, p.heads, 2);
    switch (std::max(1, p.bs * D / 2048)) {
        case 1: kv_write_kernel<T, D, 1><<<grid, 32, 0, s>>>(p); break;
        case 2: kv_write_kernel<T, D, 2><<<grid, 64, 0, s>>>(p); break;
        case 4: kv_write_kernel<T, D, 4><<<grid, 128, 0, s>>>(p); break;
        default: if constexpr (D == 128) kv_write_kernel<T, D, 8><<<grid, 256, 0, s>>>(p);
    }
    B200_CUDA_OK(cudaGetLastError());
    count_launch();
    return 0;
}

bool aligned16(const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; }

}  // namespace

int kv_block_shift(int block_size) {
    switch (block_size) { case 16: return 4; case 32: return 5; case 64: return 6; case 128: return 7; default: return -1; }
}

}  // namespace b200

using namespace b200;

extern "C" {

int pyc_b200_kv_plan(const pyc_b200_kv_plan_args* a, void* stream) {
    if (!a || !a->context_lens || !a->new_lens || !a->free_blocks || !a->free_count || !a->block_table || !a->query_start || !a->seq_lens ||
        !a->slot_map || !a->positions || !a->token_request || !a->result) { set_error("kv plan: NULL argument"); return -1; }
    const int shift = kv_block_shift(a->block_size);
    if (shift < 0) { set_error("kv plan: block_size %d is not 16, 32, 64 or 128", a->block_size); return -1; }
    if (a->requests < 1 || a->requests > PLAN_MAX_REQUESTS) { set_error("kv plan: %d requests (1 .. %d)", a->requests, PLAN_MAX_REQUESTS); return -1; }
    if (a->seq_lens == a->context_lens || a->seq_lens == a->new_lens) { set_error("kv plan: seq_lens must not be context_lens or new_lens"); return -1; }
    if (a->num_blocks < 1 || a->max_blocks < 1 || a->max_tokens < 1) { set_error("kv plan: num_blocks, max_blocks and max_tokens must be positive"); return -1; }
    if (static_cast<long long>(a->max_blocks) * a->block_size > INT_MAX) { set_error("kv plan: max_blocks * block_size exceeds 2^31 - 1 tokens"); return -1; }
    const size_t smem = static_cast<size_t>(a->requests) * 2 * sizeof(int);
    if (smem > 40 * 1024) B200_CUDA_OK(cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PLAN_MAX_REQUESTS * 8));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    // one CTA up to 4 entries per thread, then a cluster of the portable size
    attr.val.clusterDim.x = a->max_tokens > 4 * PLAN_THREADS ? 8 : 1; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(attr.val.clusterDim.x); cfg.blockDim = dim3(PLAN_THREADS); cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream); cfg.attrs = &attr; cfg.numAttrs = 1;
    B200_CUDA_OK(cudaLaunchKernelEx(&cfg, kv_plan_kernel, *a, shift));
    count_launch();
    return 0;
}

int pyc_b200_kv_release(int requests, int block_size, int num_blocks, int max_blocks, const int* finished, int* context_lens, int* block_table,
                        int* free_blocks, int* free_count, void* stream) {
    if (!finished || !context_lens || !block_table || !free_blocks || !free_count) { set_error("kv release: NULL argument"); return -1; }
    const int shift = kv_block_shift(block_size);
    if (shift < 0) { set_error("kv release: block_size %d is not 16, 32, 64 or 128", block_size); return -1; }
    if (requests < 1 || requests > PLAN_MAX_REQUESTS) { set_error("kv release: %d requests (1 .. %d)", requests, PLAN_MAX_REQUESTS); return -1; }
    if (num_blocks < 1 || max_blocks < 1) { set_error("kv release: num_blocks and max_blocks must be positive"); return -1; }
    const size_t smem = static_cast<size_t>(requests) * sizeof(int);
    if (smem > 40 * 1024) B200_CUDA_OK(cudaFuncSetAttribute(kv_release_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PLAN_MAX_REQUESTS * 4));
    kv_release_kernel<<<1, PLAN_THREADS, smem, static_cast<cudaStream_t>(stream)>>>(requests, block_size, shift, num_blocks, max_blocks, finished, context_lens,
                                                                                    block_table, free_blocks, free_count);
    B200_CUDA_OK(cudaGetLastError());
    count_launch();
    return 0;
}

int pyc_b200_kv_write(const pyc_b200_kv_write_args* a, void* stream) {
    if (!a || !a->k || !a->v || !a->slot_map || !a->k_cache || !a->v_cache || !a->k_scale || !a->v_scale) { set_error("kv write: NULL argument"); return -1; }
    if (a->dtype != PYC_DTYPE_BF16 && a->dtype != PYC_DTYPE_F16) { set_error("kv write: keys and values must be bf16 or f16"); return -1; }
    const int shift = kv_block_shift(a->block_size);
    if (shift < 0) { set_error("kv write: block_size %d is not 16, 32, 64 or 128", a->block_size); return -1; }
    if (a->head_dim != 64 && a->head_dim != 128) { set_error("kv write: head_dim %d is not 64 or 128", a->head_dim); return -1; }
    if (a->tokens < 1 || a->kv_heads < 1 || a->kv_heads > 65535 || a->num_blocks < 1) { set_error("kv write: tokens, kv_heads (up to 65535) and num_blocks must be positive"); return -1; }
    const size_t row = static_cast<size_t>(a->kv_heads) * a->head_dim;
    const size_t ks = a->k_stride ? a->k_stride : row, vs = a->v_stride ? a->v_stride : row;
    if (ks < row || vs < row || ks % 8 || vs % 8) { set_error("kv write: row strides must be multiples of 8 and at least kv_heads * head_dim"); return -1; }
    if (!aligned16(a->k) || !aligned16(a->v) || !aligned16(a->k_cache) || !aligned16(a->v_cache)) { set_error("kv write: pointers must be 16-byte aligned"); return -1; }
    KvWriteParams p;
    p.x[0] = a->k; p.x[1] = a->v; p.stride[0] = ks; p.stride[1] = vs;
    p.cache[0] = static_cast<uint8_t*>(a->k_cache); p.cache[1] = static_cast<uint8_t*>(a->v_cache);
    p.scale[0] = a->k_scale; p.scale[1] = a->v_scale;
    p.slots = a->slot_map; p.tokens = a->tokens; p.heads = a->kv_heads; p.bs = a->block_size; p.shift = shift; p.num_blocks = a->num_blocks;
    // Tokens per CTA: 1 where there are few (every token may be a run of its own), up to a block where there are many (then most
    // tokens do not begin a run), as long as every SM keeps 32 CTAs to choose from.
    const long long units = 2ll * a->tokens * a->kv_heads / (static_cast<long long>(sm_count()) * 32);
    p.group = 1;
    while (p.group < a->block_size && p.group * 2 <= units) p.group *= 2;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->dtype == PYC_DTYPE_BF16) return a->head_dim == 128 ? launch_kv_write<__nv_bfloat16, 128>(p, s) : launch_kv_write<__nv_bfloat16, 64>(p, s);
    return a->head_dim == 128 ? launch_kv_write<__half, 128>(p, s) : launch_kv_write<__half, 64>(p, s);
}

}  // extern "C"
