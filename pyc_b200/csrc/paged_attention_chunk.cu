// Attention over the 8-bit paged cache for many query rows per key head: chunks of prompts, bound by the products.  Items,
// stretches, split items and their joining are those of paged_attention.cuh; an item's tile has 128 rows (queries times query
// heads of a key head), a unit 64 keys.
//
// 256 threads per CTA, two CTAs per SM, so that one's tensor-core work passes beside the other's softmax:
//   warp 0      TMEM owner and single-thread MMA issuer
//                 S[n&1] = Q K_n^T     128 x 64 x D    (tcgen05, f16, S in TMEM, two buffers)
//                 O     += P_n V_n     128 x D x 64    (P_n from TMEM, where S_n was; V as MN-major operand)
//   warps 1-3   bring the blocks in: 16-byte loads of e4m3 codes, f16 (exact, two codes per conversion) into the 128-byte-swizzled
//               operand layout, the next block's loads under way meanwhile.  tcgen05 has no product of e4m3 with 16-bit
//               operands; splitting the queries into e4m3 terms, as the kernel for few rows does, would spare the keys'
//               conversion but not the values', and 128 rows share each conversion here
//   warps 4-7   softmax, one query row per thread; they make the queries' operand first and write the result last
// Precision is that of paged_attention.cu: queries scaled per row by a power of two and then rounded to f16, which loses
// what lies below 2^-24 of the row's largest; p' = 2^(score + log2 vs - m) as f16, the softmax's weight sum p' / vs in f32.
// Values that some row must not see are zero in the operand where they are NaN; the rows that do see one get their NaN at the
// end (nan_key: the first key, of those that not every row sees, with a NaN in a column).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

#include "internal.h"
#include "paged_attention.cuh"
#include "paged_attention_chunk.h"
#include "ptx_sm100.cuh"

namespace b200 {
namespace {

constexpr int BQ = 128, BK = 64;
constexpr int THREADS = 256, CONVERTERS = 96;

template <int D>
struct ChunkSmem {
    static constexpr int Q_BYTES = BQ * D * 2, KV_TILE = BK * D * 2;
    static constexpr int K_OFF = Q_BYTES, V_OFF = K_OFF + 2 * KV_TILE;
    static constexpr int INFO_OFF = V_OFF + 2 * KV_TILE;                 // float4 [4][4]: per block (mod 4) and 16 keys
    static constexpr int NAN_OFF = INFO_OFF + 256;                       // int [D]
    static constexpr int BAR_OFF = NAN_OFF + D * 4;                      // q | k full, empty | v full, empty | s full | p full (2 each) | pv done | o done
    static constexpr int NUM_BARS = 16;
    static constexpr int SHARES_OFF = BAR_OFF + NUM_BARS * 8 + 16;       // behind the barriers: TMEM address, failure flag
    static constexpr int SPLIT_OFF = SHARES_OFF + sizeof(PagedShares);
    static constexpr int BYTES = SPLIT_OFF + 2 * sizeof(PagedCursor) + 16;
    static_assert((BYTES + 1024) * 2 <= 228 * 1024, "two CTAs per SM");
    static_assert(2 * 16 * (1 + 320) * 4 <= INFO_OFF, "the join's scratch: 16 rows of up to 320 parts");
};

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
template <typename T> __device__ __forceinline__ float2 wide2(uint32_t w);
template <> __device__ __forceinline__ float2 wide2<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
template <> __device__ __forceinline__ float2 wide2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// 0x80 in each byte that is a NaN code.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 2)
paged_chunk_kernel(const __grid_constant__ PagedParams p, const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache) {
    using SM = ChunkSmem<D>;
    constexpr int HALVES = D / 64, Q_SLAB = BQ * 128, KV_SLAB = BK * 128;
    constexpr uint32_t IDESC_QK = make_idesc(0, 0, 0, 0, BQ, BK), IDESC_PV = make_idesc(0, 0, 0, 1, BQ, D);
    constexpr uint32_t TMEM_COLS = 256, O_COL = 128;                         // S0 @0, S1 @64, O @128
    extern __shared__ __align__(1024) uint8_t smem[];
    float4* info = reinterpret_cast<float4*>(smem + SM::INFO_OFF);
    int* nan_key = reinterpret_cast<int*>(smem + SM::NAN_OFF);
    uint64_t* bar_mem = reinterpret_cast<uint64_t*>(smem + SM::BAR_OFF);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_mem + SM::NUM_BARS);
    PagedShares& shares = *reinterpret_cast<PagedShares*>(smem + SM::SHARES_OFF);
    PagedCursor (&split)[2] = *reinterpret_cast<PagedCursor (*)[2]>(smem + SM::SPLIT_OFF);
    int (&is_split)[2] = *reinterpret_cast<int (*)[2]>(smem + SM::SPLIT_OFF + 2 * sizeof(PagedCursor));
    int* flags = reinterpret_cast<int*>(smem + SM::SPLIT_OFF + 2 * sizeof(PagedCursor) + 8);
    const uint32_t bar0 = smem_u32(bar_mem);
    const uint32_t q_full = bar0, k_full = bar0 + 8, k_empty = bar0 + 24, v_full = bar0 + 40, v_empty = bar0 + 56, s_full = bar0 + 72, p_full = bar0 + 88, pv_done = bar0 + 104, o_done = bar0 + 112;
    const uint32_t sQ = smem_u32(smem), sK = sQ + SM::K_OFF, sV = sQ + SM::V_OFF;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        mbar_init(q_full, 4);
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full + 8 * i, CONVERTERS / 32); mbar_init(k_empty + 8 * i, 1);
            mbar_init(v_full + 8 * i, CONVERTERS / 32); mbar_init(v_empty + 8 * i, 1);
            mbar_init(s_full + 8 * i, 1); mbar_init(p_full + 8 * i, 4);
        }
        mbar_init(pv_done, 1); mbar_init(o_done, 1);
        fence_barrier_init();
        fence_proxy_async();
        is_split[0] = is_split[1] = 0;
    }
    PagedCursor c;
    const bool busy = paged_begin<THREADS, BQ, BK>(p, c, shares);
    __syncthreads();
    if (!busy) return;
    if (warp == 0) { tmem_alloc(smem_u32(tmem_slot), TMEM_COLS); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
    uint32_t n = 0;                                      // blocks before this item: every role counts them alike
    uint32_t items = 0;

    for (;; ++items) {
        const int j0 = c.from(), j1 = c.to(), blocks = j1 - j0;
        const int row0 = c.t * BQ, rows = min(BQ, c.q.rows - row0);
        const int kend = paged_tile_end<BQ>(p, c.q, c.t);
        const int all_see = paged_limit(p, c.q, row0 / p.group);             // keys that every row sees
        if (threadIdx.x < D) nan_key[threadIdx.x] = INT_MAX;
        __syncthreads();
        bool ok = true;

        if (warp == 0) {
            if (lane == 0) {
                constexpr uint32_t HI = smem_desc_hi_sw128(1024);
                const uint32_t q_lo = smem_desc_lo(sQ, 16), k_lo0 = smem_desc_lo(sK, 16), v_lo0 = smem_desc_lo(sV, KV_SLAB);
                auto issue_qk = [&](uint32_t b) {                            // S[b&1] = Q K_b^T
                    const uint32_t st = b & 1, k_lo = k_lo0 + st * (SM::KV_TILE >> 4);
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks)
                        umma_f16(tmem_base + st * BK, smem_desc_join(q_lo + (((ks / 4) * Q_SLAB + (ks % 4) * 32) >> 4), HI),
                                 smem_desc_join(k_lo + (((ks / 4) * KV_SLAB + (ks % 4) * 32) >> 4), HI), IDESC_QK, ks != 0);
                    umma_commit(s_full + 8 * st);
                    umma_commit(k_empty + 8 * st);
                };
                ok = mbar_wait(q_full, items & 1, p.status, 0x63);
                tc_fence_after();
                for (int i = 0; i < 2 && i < blocks && ok; ++i) {            // two score blocks in flight before the first P arrives
                    const uint32_t b = n + i;
                    if (!mbar_wait(k_full + 8 * (b & 1), (b >> 1) & 1, p.status, 0x64)) { ok = false; break; }
                    tc_fence_after();
                    issue_qk(b);
                }
                for (int i = 0; i < blocks && ok; ++i) {
                    const uint32_t b = n + i, st = b & 1, par = (b >> 1) & 1;
                    if (!mbar_wait(v_full + 8 * st, par, p.status, 0x65)) { ok = false; break; }
                    if (!mbar_wait(p_full + 8 * st, par, p.status, 0x66)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t v_lo = v_lo0 + st * (SM::KV_TILE >> 4);
#pragma unroll
                    for (int ks = 0; ks < BK / 16; ++ks)
                        umma_f16_ts(tmem_base + O_COL, tmem_base + st * BK + ks * 8, smem_desc_join(v_lo + ks * (2048 >> 4), HI), IDESC_PV, (i | ks) != 0 ? 1u : 0u);
                    umma_commit(v_empty + 8 * st);
                    umma_commit(pv_done);
                    if (i + 1 == blocks) umma_commit(o_done);
                    if (i + 2 < blocks) {                                    // S[st] is free once this P V is in the pipe ahead
                        const uint32_t b2 = b + 2;
                        if (!mbar_wait(k_full + 8 * (b2 & 1), (b2 >> 1) & 1, p.status, 0x67)) { ok = false; break; }
                        tc_fence_after();
                        issue_qk(b2);
                    }
                }
            }
            __syncwarp();
        } else if (warp < 4) {
            // ---- codes to f16 operands.  Chunk x of a block: 16 codes of token x / (D / 16), from column 16 * (x % (D / 16)).
            constexpr int PER_ROW = D / 16, CHUNKS = BK * PER_ROW, LOADS = (CHUNKS + CONVERTERS - 1) / CONVERTERS;
            const int ct = threadIdx.x - 32;
            const int* table = p.table + static_cast<size_t>(c.r) * p.max_blocks;
            uint4 kx[LOADS], vx[LOADS];
            // lane g < 4 of each warp: block and scales of the block's 16-token group g
            auto block_of = [&](int j) {
                const int key = j * BK + lane * 16;
                int id = -1;
                if (lane < 4 && j < j1 && key < kend) id = __ldg(table + (key >> p.shift));
                return static_cast<unsigned>(id) < static_cast<unsigned>(p.num_blocks) ? id : -1;
            };
            auto load = [&](const uint8_t* cache, int j, int id, uint4 (&to)[LOADS]) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const int x = ct + i * CONVERTERS, t = x / PER_ROW, key = j * BK + t;
                    const int mine = __shfl_sync(0xffffffffu, id, (t >> 4) & 3);
                    to[i] = make_uint4(0, 0, 0, 0);
                    if (x < CHUNKS && mine >= 0 && key < kend)
                        to[i] = __ldg(reinterpret_cast<const uint4*>(cache + ((static_cast<size_t>(mine) * p.kv_heads + c.h) * p.block_size + (key & (p.block_size - 1))) * D) + x % PER_ROW);
                }
            };
            auto store = [&](uint32_t tile, const uint4 (&from)[LOADS]) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const int x = ct + i * CONVERTERS, t = x / PER_ROW, col = (x % PER_ROW) * 2;      // in 16-byte chunks of 8 f16
                    if (x >= CHUNKS) break;
                    uint32_t h[8];
                    e4m3x4_to_f16x4(from[i].x, h[0], h[1]); e4m3x4_to_f16x4(from[i].y, h[2], h[3]);
                    e4m3x4_to_f16x4(from[i].z, h[4], h[5]); e4m3x4_to_f16x4(from[i].w, h[6], h[7]);
                    const uint32_t line = tile + (col >> 3) * KV_SLAB + t * 128, sw = t & 7;
                    sts128(line + (((col & 7) ^ sw) << 4), h[0], h[1], h[2], h[3]);
                    sts128(line + ((((col & 7) + 1) ^ sw) << 4), h[4], h[5], h[6], h[7]);
                }
            };
            int id = block_of(j0);
            load(k_cache, j0, id, kx);
            load(v_cache, j0, id, vx);
            for (int j = j0; j < j1 && ok; ++j) {
                const uint32_t b = n + (j - j0), st = b & 1, par = ((b >> 1) & 1) ^ 1;
                const int id_next = block_of(j + 1);
                float ks = 0.0f, vs = 1.0f;
                if (id >= 0) {
                    const size_t at = static_cast<size_t>(id) * p.kv_heads + c.h;
                    ks = paged_clamp_scale(__ldg(p.k_scale + at)); vs = paged_clamp_scale(__ldg(p.v_scale + at));
                }
                ok = __all_sync(0xffffffffu, mbar_wait(k_empty + 8 * st, par, p.status, 0x68));
                if (!ok) break;
                if (warp == 1 && lane < 4) info[(b & 3) * 4 + lane] = make_float4(ks, log2f(vs), 1.0f / vs, 0.0f);
                store(sK + st * SM::KV_TILE, kx);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(k_full + 8 * st);
                load(k_cache, j + 1, id_next, kx);
                if ((j + 1) * BK > all_see) {
                    // keys that some row does not see: NaN values leave the operand, and the first key with one is kept for each column
#pragma unroll
                    for (int i = 0; i < LOADS; ++i) {
                        const int x = ct + i * CONVERTERS, key = j * BK + x / PER_ROW;
                        uint32_t w[4] = {vx[i].x, vx[i].y, vx[i].z, vx[i].w};
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            const uint32_t z = nan_bytes(w[y]);
                            if (z != 0 && x < CHUNKS) {
                                for (int e = 0; e < 4; ++e) if (z & (0x80u << (8 * e))) atomicMin(nan_key + (x % PER_ROW) * 16 + y * 4 + e, key);
                                w[y] &= ~((z >> 7) * 0xffu);
                            }
                        }
                        vx[i] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                ok = __all_sync(0xffffffffu, mbar_wait(v_empty + 8 * st, par, p.status, 0x69));
                if (!ok) break;
                store(sV + st * SM::KV_TILE, vx);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(v_full + 8 * st);
                load(v_cache, j + 1, id_next, vx);
                id = id_next;
            }
        } else {
            const int wq = warp & 3, row = wq * 32 + lane;
            const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(wq * 32) << 16);
            const int token = (row0 + min(row, rows - 1)) / p.group, head = c.h * p.group + (row0 + min(row, rows - 1) - token * p.group);
            const int lim = paged_limit(p, c.q, token);
            // ---- this thread's query row, scaled to [1, 2) by a power of two, as f16 operand
            float qs;
            bool finite = true;                                              // one that is not becomes zeros, and NaN at the end if it sees a key
            {
                const T* src = static_cast<const T*>(p.q) + (static_cast<size_t>(c.q.start) + token) * p.q_stride + static_cast<size_t>(head) * D;
                float amax = 0.0f;
#pragma unroll 4
                for (int i = 0; i < D / 8; ++i) {
                    const uint4 u = __ldg(reinterpret_cast<const uint4*>(src) + i);
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const float2 f = wide2<T>(w[y]);
                        amax = max3(amax, fabsf(f.x), fabsf(f.y));
                        finite &= fabsf(f.x) < INFINITY && fabsf(f.y) < INFINITY;
                    }
                }
                // at the ends of the range, where 2^e or 2^-e would be subnormal, to [0, 4)
                const int e = amax > 0.0f && finite ? min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, -126), 126) : 0;
                const float down = exp2_int(-e);
                qs = exp2_int(e) * p.scale_log2;
#pragma unroll 4
                for (int i = 0; i < D / 8; ++i) {
                    const uint4 u = __ldg(reinterpret_cast<const uint4*>(src) + i);
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
                    uint32_t h[4];
#pragma unroll
                    for (int y = 0; y < 4; ++y) { const float2 f = wide2<T>(w[y]); h[y] = finite ? pack_f16(f.x * down, f.y * down) : 0u; }
                    sts128(sQ + (i >> 3) * Q_SLAB + row * 128 + (((i & 7) ^ (row & 7)) << 4), h[0], h[1], h[2], h[3]);
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            }
            float m = -INFINITY, l = 0.0f;
            const int warp_sees = __shfl_sync(0xffffffffu, lim, 0);          // keys that every row of the warp sees
            for (int i = 0; i < blocks && ok; ++i) {
                const uint32_t b = n + i, st = b & 1, s_addr = lane_addr + st * BK;
                if (!mbar_wait(s_full + 8 * st, (b >> 1) & 1, p.status, 0x6a)) { ok = false; break; }
                tc_fence_after();
                const int k0 = (j0 + i) * BK;
                uint32_t r[64];
                tmem_ld_32x32(s_addr, reinterpret_cast<uint32_t (&)[32]>(r[0]));
                tmem_ld_32x32(s_addr + 32, reinterpret_cast<uint32_t (&)[32]>(r[32]));
                float4 in[4];
#pragma unroll
                for (int g = 0; g < 4; ++g) in[g] = info[(b & 3) * 4 + g];
                tmem_ld_wait();
                const bool gone = in[0].x == 0.0f || in[1].x == 0.0f || in[2].x == 0.0f || in[3].x == 0.0f;
                if (k0 + BK > warp_sees || gone) {
#pragma unroll
                    for (int x = 0; x < 64; ++x) if (k0 + x >= lim || in[x >> 4].x == 0.0f) r[x] = 0xff800000u;      // -inf
                }
                float f[4], m_blk = -INFINITY;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float mx = -INFINITY, my = -INFINITY;
#pragma unroll
                    for (int x = 0; x < 16; x += 4) {
                        mx = max3(mx, __uint_as_float(r[g * 16 + x]), __uint_as_float(r[g * 16 + x + 1]));
                        my = max3(my, __uint_as_float(r[g * 16 + x + 2]), __uint_as_float(r[g * 16 + x + 3]));
                    }
                    f[g] = in[g].x > 0.0f ? qs * in[g].x : 1.0f;             // of a masked group: -inf stays -inf
                    m_blk = fmaxf(m_blk, fmaf(fmaxf(mx, my), f[g], in[g].y));
                }
                // the reference moves only when a score exceeds it by more than 2^8 (p' stays below f16's largest; sums are f32)
                const float m_new = fmaxf(m, m_blk);
                const bool move = m_new > m + 8.0f;
                const float m_ref = move ? m_new : m;
                const float m_use = m_ref == -INFINITY ? 0.0f : m_ref;
                const float alpha = move ? ex2_approx(m - m_use) : 1.0f;
                l *= alpha;
                m = m_ref;
                uint32_t packed[32];
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const unsigned long long f2 = f32x2_splat(f[g]), d2 = f32x2_splat(in[g].y - m_use);
                    unsigned long long l2 = 0ull;                            // (0, 0)
#pragma unroll
                    for (int x = 0; x < 16; x += 2) {
                        float a0, a1;
                        f32x2_unpack(f32x2_fma(f32x2_pack(__uint_as_float(r[g * 16 + x]), __uint_as_float(r[g * 16 + x + 1])), f2, d2), a0, a1);
                        a0 = ex2_approx(a0); a1 = ex2_approx(a1);
                        l2 = f32x2_add(l2, f32x2_pack(a0, a1));
                        packed[g * 8 + x / 2] = pack_f16(a0, a1);
                    }
                    float l0, l1;
                    f32x2_unpack(l2, l0, l1);
                    l = fmaf(l0 + l1, in[g].z, l);
                }
                // O is touched only when some row of the warp moved its reference, and only then must the previous P V have finished
                // (the one before it has, for this block's scores came behind it, and this block's cannot: the parity says which)
                if (i > 0 && __any_sync(0xffffffffu, move)) {
                    if (!mbar_wait(pv_done, (b - 1) & 1, p.status, 0x6b)) { ok = false; break; }
                    tc_fence_after();
#pragma unroll 1
                    for (int x = 0; x < D / 32; ++x) {
                        uint32_t o[32];
                        tmem_ld_32x32(lane_addr + O_COL + x * 32, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * alpha);
                        tmem_st_32x32(lane_addr + O_COL + x * 32, o);
                    }
                }
                tmem_st_32x32(s_addr, packed);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 8 * st);
            }
            // the last P V has a barrier of its own, one completion per item: this warp may come to it when any number have completed
            if (ok) ok = mbar_wait(o_done, items & 1, p.status, 0x6c);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
                tc_fence_after();
                const bool whole = j0 == 0 && j1 == c.units;
                float* part = p.partials + (static_cast<size_t>(blockIdx.x) * 2 + (j0 == 0 ? 1 : 0)) * (static_cast<size_t>(BQ) * (D + 2));
                const float ref = m == -INFINITY ? 0.0f : m;
                if (!finite && l > 0.0f) l = __int_as_float(0x7fffffff);
#pragma unroll 1
                for (int x = 0; x < D / 32; ++x) {
                    uint32_t r[32];
                    tmem_ld_32x32(lane_addr + O_COL + x * 32, r);
                    tmem_ld_wait();
                    if (row < rows) {
#pragma unroll
                        for (int y = 0; y < 32; y += 8) {
                            float v[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                v[e] = l == 0.0f ? 0.0f : __uint_as_float(r[y + e]);      // no key seen: whatever the products left
                                if (nan_key[x * 32 + y + e] < lim) v[e] = __int_as_float(0x7fffffff);
                            }
                            if (whole) paged_finish<T, D>(p, c, row0 + row, x * 32 + y, v, ref, l);
                            else {
                                float* dst = part + row * D + x * 32 + y;
                                __stcg(reinterpret_cast<float4*>(dst), make_float4(v[0], v[1], v[2], v[3]));
                                __stcg(reinterpret_cast<float4*>(dst + 4), make_float4(v[4], v[5], v[6], v[7]));
                            }
                        }
                    }
                    __syncwarp();
                }
                if (!whole && row < rows) { __stcg(part + BQ * D + row, m); __stcg(part + BQ * (D + 1) + row, l); }
            }
            tc_fence_before();
        }
        n += blocks;
        const bool whole = j0 == 0 && j1 == c.units;
        if (!whole && threadIdx.x == 0) { split[j0 == 0 ? 1 : 0] = c; is_split[j0 == 0 ? 1 : 0] = 1; }
        // the next item when every role has left this one: Q, S, O and the counters are free.  A role whose wait ran out ends the CTA's work.
        if (__syncthreads_or(!ok)) break;
        tc_fence_after();
        if (!paged_next<BQ, BK>(p, c)) break;
    }
    __syncthreads();
    if (*reinterpret_cast<volatile int*>(p.status) != ST_OK) for (int i = 0; i < 2000; ++i) __nanosleep(1000);       // let what is in flight land
    tc_fence_after();
    if (warp == 0) tmem_dealloc(tmem_base, TMEM_COLS);
    paged_announce<T, D, THREADS, BQ>(p, shares, split, is_split, flags, reinterpret_cast<float*>(smem));
}

template <typename T, int D>
int launch(const PagedParams& p, const void* k_cache, const void* v_cache, cudaStream_t s) {
    auto kernel = paged_chunk_kernel<T, D>;
    B200_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ChunkSmem<D>::BYTES));
    kernel<<<paged_chunk_ctas(), THREADS, ChunkSmem<D>::BYTES, s>>>(p, static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache));
    B200_CUDA_OK(cudaGetLastError());
    count_launch();
    return 0;
}

}  // namespace

int paged_chunk_ctas() { return std::min(sm_count() * 2, 320); }
size_t paged_chunk_partial_bytes(int head_dim) { return static_cast<size_t>(paged_chunk_ctas()) * 2 * BQ * (head_dim + 2) * sizeof(float); }

int launch_paged_chunk(pyc_dtype dtype, int head_dim, PagedParams p, const void* k_cache, const void* v_cache, cudaStream_t s) {
    // an item's queries, first blocks and result take about as long as ten units of 64 keys (0.5 us each with two CTAs on the SM)
    p.cost = 10; p.unsplit = 16;
    if (dtype == PYC_DTYPE_F16) return head_dim == 128 ? launch<__half, 128>(p, k_cache, v_cache, s) : launch<__half, 64>(p, k_cache, v_cache, s);
    return head_dim == 128 ? launch<__nv_bfloat16, 128>(p, k_cache, v_cache, s) : launch<__nv_bfloat16, 64>(p, k_cache, v_cache, s);
}

}  // namespace b200
