// Attention over the 8-bit paged cache for many query rows per key head: chunks of prompts, bound by products and softmax.  Items,
// stretches, split items and their joining are those of paged_attention.cuh; an item has two tiles of 128 rows (queries times
// query heads of a key head), a unit 64 keys.
//
// One CTA per SM, 16 warps:
//   warps 0, 1   one thread each issues the products of one tile t (warp 0 owns TMEM)
//                  S_t[n&1] = Q_t K_n^T     128 x 64 x D    (tcgen05, f16, S in TMEM, two buffers per tile)
//                  O_t     += P_n V_n       128 x D x 64    (P_n from TMEM, where S_n was; V as MN-major operand)
//   warp 2       brings the blocks' codes in (bulk copies, RAW stages), with the scales of their 16-token groups
//   warp 3       idle: softmax warps have to begin at a multiple of four, for the TMEM lanes that they may read
//   warps 4-7    codes to f16 operands (exact, two codes per conversion) in the 128-byte-swizzled layout.  tcgen05 has no product of
//                e4m3 with 16-bit operands; splitting the queries into e4m3 terms, as the kernel for few rows does, would spare the
//                keys' conversion but not the values', and 256 rows share each conversion here
//   warps 8-15   softmax, one query row per thread; they make the next item's operand before they write an item's result
// The roles meet at mbarriers only and walk the items each on its own, so that the next item's blocks come in, are converted and
// multiplied while the softmax warps write this one's result.
//
// Measured: 4 requests with chunks of 2048 queries behind up to 5000 keys (8 x 4 heads of 128, bf16, 0.254 TFLOP) take 347 us = 732
// TFLOP/s; 8 prompts of 1000 tokens with nothing before them 177 us, of which 7 items per CTA take about 5 us each at their ends.
// Of 2700 clocks per block of 64 keys and both tiles a softmax warp computes for 2200 (two warps share an XU whose
// exponentials alone take 1024, and each goes load, maximum, exponentials, store in turn), the issuing threads wait for it 1300;
// neither products (8 us), conversions (16 us) nor half of the exponentials (22 us) left out changed much.  Ways here: one tile per CTA, two
// CTAs per SM, converters that load codes themselves 780 us; two tiles that share conversions 627; queries, results and operands in 16-byte
// pieces without bank conflicts 601; descriptors in uniform registers (an elected lane) 415; an issuing warp per tile instead of one for
// both 381; the join, a row per thread and sums in 512-byte pieces, 347.
//
// Precision is that of paged_attention.cu: queries scaled per row by a power of two and then rounded to f16, which loses
// what lies below 2^-24 of the row's largest; p' = 2^(score + log2 vs - m) as f16, the softmax's weight sum p' / vs in f32.
// Values that some row must not see are zero in the operand where they are NaN; where that happened, the rows look the NaN
// that they do see up in the cache at the item's end.
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

constexpr int BQ = 128, TILES = 2, ROWS = BQ * TILES, BK = 64;
constexpr int COPY_WARP = 2, CONVERT_WARP = 4, CONVERT_WARPS = 4, SOFTMAX_WARP = 8;     // the first TILES warps issue the products
constexpr int CONVERTERS = CONVERT_WARPS * 32, THREADS = (SOFTMAX_WARP + 4 * TILES) * 32;
constexpr int RING = 16;                                 // entries of what is kept per block and per item: more than the roles can be apart

template <int D>
struct ChunkSmem {
    static constexpr int RAW = 4;                                        // stages of codes
    static constexpr int Q_BYTES = BQ * D * 2, KV_TILE = BK * D * 2, RAW_TILE = BK * D;
    static constexpr int K_OFF = TILES * Q_BYTES, V_OFF = K_OFF + 2 * KV_TILE, RAW_OFF = V_OFF + 2 * KV_TILE;
    static constexpr int OUT_OFF = RAW_OFF + RAW * 2 * RAW_TILE;         // per softmax warp 32 rows of 32 results, on their way out
    static constexpr int INFO_OFF = OUT_OFF + 4 * TILES * 2048;          // float4 [RING][4]: per block and 16 keys
    static constexpr int NAN_OFF = INFO_OFF + RING * 64;                 // int [RING]: per item, whether a NaN value was left out
    static constexpr int BAR_OFF = NAN_OFF + RING * 4;
    static constexpr int NUM_BARS = 2 * RAW + 8 + 7 * TILES;             // raw full, empty | k full, empty, v full, empty (2 each) | per tile: q, s full (2), p full (2), pv done, o done
    static constexpr int SHARES_OFF = BAR_OFF + NUM_BARS * 8 + 16;       // behind the barriers: the TMEM address
    static constexpr int SPLIT_OFF = SHARES_OFF + sizeof(PagedShares);
    static constexpr int BYTES = SPLIT_OFF + 2 * sizeof(PagedCursor) + 16;
    static_assert(BYTES + 1024 <= 228 * 1024 && SHARES_OFF % 8 == 0, "shared memory of an SM");
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
template <typename T> struct Bf16 { static constexpr bool value = false; };
template <> struct Bf16<__nv_bfloat16> { static constexpr bool value = true; };
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// 0x80 in each byte that is a NaN code.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// True in one lane of a converged warp; unlike a comparison of the lane number, it lets the compiler keep what the lane computes in
// uniform registers, where tcgen05.mma takes its descriptors from.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
// Untiled copy of `bytes` (a multiple of 16; both addresses 16-byte aligned), counted on `bar`.
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 1)
paged_chunk_kernel(const __grid_constant__ PagedParams p, const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache) {
    using SM = ChunkSmem<D>;
    constexpr int Q_SLAB = BQ * 128, KV_SLAB = BK * 128, RAW = SM::RAW;
    constexpr uint32_t IDESC_QK = make_idesc(0, 0, 0, 0, BQ, BK), IDESC_PV = make_idesc(0, 0, 0, 1, BQ, D);
    constexpr uint32_t TMEM_COLS = 512, TILE_COLS = 256, O_COL = 128;        // per tile: S0 @0, S1 @64, O @128
    extern __shared__ __align__(1024) uint8_t smem[];
    float4* info = reinterpret_cast<float4*>(smem + SM::INFO_OFF);
    int* left_out = reinterpret_cast<int*>(smem + SM::NAN_OFF);
    uint64_t* bar_mem = reinterpret_cast<uint64_t*>(smem + SM::BAR_OFF);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_mem + SM::NUM_BARS);
    PagedShares& shares = *reinterpret_cast<PagedShares*>(smem + SM::SHARES_OFF);
    PagedCursor (&split)[2] = *reinterpret_cast<PagedCursor (*)[2]>(smem + SM::SPLIT_OFF);
    int (&is_split)[2] = *reinterpret_cast<int (*)[2]>(smem + SM::SPLIT_OFF + 2 * sizeof(PagedCursor));
    int* flags = reinterpret_cast<int*>(smem + SM::SPLIT_OFF + 2 * sizeof(PagedCursor) + 8);
    const uint32_t raw_full = smem_u32(bar_mem), raw_empty = raw_full + 8 * RAW, k_full = raw_empty + 8 * RAW, k_empty = k_full + 16, v_full = k_full + 32, v_empty = k_full + 48;
    const uint32_t tile_bars = k_full + 64;              // 7 per tile
    auto q_full = [&](int t) { return tile_bars + t * 56; };
    auto s_full = [&](int t, uint32_t st) { return tile_bars + t * 56 + 8 + 8 * st; };
    auto p_full = [&](int t, uint32_t st) { return tile_bars + t * 56 + 24 + 8 * st; };
    auto pv_done = [&](int t) { return tile_bars + t * 56 + 40; };
    auto o_done = [&](int t) { return tile_bars + t * 56 + 48; };
    const uint32_t sQ = smem_u32(smem), sK = sQ + SM::K_OFF, sV = sQ + SM::V_OFF, sR = sQ + SM::RAW_OFF;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < RAW; ++i) { mbar_init(raw_full + 8 * i, 1); mbar_init(raw_empty + 8 * i, CONVERT_WARPS); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full + 8 * i, CONVERT_WARPS); mbar_init(k_empty + 8 * i, TILES);
            mbar_init(v_full + 8 * i, CONVERT_WARPS); mbar_init(v_empty + 8 * i, TILES);
        }
        for (int t = 0; t < TILES; ++t) {
            mbar_init(q_full(t), 4); mbar_init(pv_done(t), 1); mbar_init(o_done(t), 1);
            for (int i = 0; i < 2; ++i) { mbar_init(s_full(t, i), 1); mbar_init(p_full(t, i), 4); }
        }
        fence_barrier_init();
        fence_proxy_async();
        is_split[0] = is_split[1] = 0;
    }
    PagedCursor c;
    const bool busy = paged_begin<THREADS, ROWS, BK>(p, c, shares);
    __syncthreads();
    if (!busy) return;
    if (warp == 0) { tmem_alloc(smem_u32(tmem_slot), TMEM_COLS); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
    uint32_t pv = 0, done = 0;                           // blocks and items before this one of this warp's tile (tile 1 has no part in items of up to 128 rows)
    bool ok = true;
    // Each role walks the items in a loop of its own.
    struct Item {
        uint32_t number, n;                              // items and blocks before this one: every role counts them alike
        int j0, j1, blocks, row0, rows, tiles, kend, all_see;
    };
    auto walk = [&](auto&& role) {
        uint32_t n = 0;
        for (uint32_t number = 0; ok; ++number) {
            Item it;
            it.number = number; it.n = n;
            it.j0 = c.from(); it.j1 = c.to(); it.blocks = it.j1 - it.j0;
            it.row0 = c.t * ROWS; it.rows = min(ROWS, c.q.rows - it.row0); it.tiles = it.rows > BQ ? 2 : 1;
            it.kend = paged_tile_end<ROWS>(p, c.q, c.t);
            it.all_see = paged_limit(p, c.q, it.row0 / p.group);             // keys that every row sees
            role(it);
            n += it.blocks;
            if (!paged_next<ROWS, BK>(p, c)) break;
        }
    };

    // A softmax warp's tile and place in it, and what it knows of the row whose score it forms next.
    const int t = (warp - SOFTMAX_WARP) >> 2, wq = warp & 3, in_tile = wq * 32 + lane;
    const uint32_t lane_addr = tmem_base + t * TILE_COLS + (static_cast<uint32_t>(wq * 32) << 16);
    float next_qs = 0.0f;                                // its scale
    bool next_finite = true;                             // a row that is not becomes zeros, and NaN at the end if it sees a key
    // The warp's 32 query rows of item x, each scaled to [1, 2) by a power of two, as f16 operand.  D / 8 lanes read one row.
    auto queries = [&](const PagedCursor& x) {
        const int row0 = x.t * ROWS, rows = min(ROWS, x.q.rows - row0);
        if (t * BQ >= rows) return;
        constexpr int LPR = D / 8, RPL = 32 / LPR, LOADS = 32 / RPL;
        const int at_row = row0 + min(t * BQ + in_tile, rows - 1), token = at_row / p.group, head = x.h * p.group + (at_row - token * p.group);
        const size_t row_at = (static_cast<size_t>(x.q.start) + token) * p.q_stride + static_cast<size_t>(head) * D;
        uint4 u[LOADS];
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            u[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + __shfl_sync(0xffffffffu, row_at, i * RPL + lane / LPR)) + lane % LPR);
        constexpr uint32_t INF = Bf16<T>::value ? 0x7f80 : 0x7c00;
        uint32_t own = 0;                                // magnitude of the thread's own row
        // at the ends of the range, where 2^e or 2^-e would be subnormal, to [0, 4)
        auto exponent = [&](uint32_t bits) {
            const float amax = wide2<T>(bits).x;
            return amax > 0.0f && bits < INF ? min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, -126), 126) : 0;
        };
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
            uint32_t bits = 0, h[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) bits = __vmaxu2(bits, w[y] & 0x7fff7fffu);
            bits = max(bits & 0xffffu, bits >> 16);
#pragma unroll
            for (int y = LPR / 2; y > 0; y >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, y));
            const float down = exp2_int(-exponent(bits));
            const uint32_t of_own = __shfl_sync(0xffffffffu, bits, (lane % RPL) * LPR);
            if (lane / RPL == i) own = of_own;
#pragma unroll
            for (int y = 0; y < 4; ++y) { const float2 f = wide2<T>(w[y]); h[y] = bits < INF ? pack_f16(f.x * down, f.y * down) : 0u; }
            const int line = wq * 32 + i * RPL + lane / LPR, piece = lane % LPR;
            sts128(sQ + t * SM::Q_BYTES + (piece >> 3) * Q_SLAB + line * 128 + (((piece & 7) ^ (line & 7)) << 4), h[0], h[1], h[2], h[3]);
        }
        next_qs = exp2_int(exponent(own)) * p.scale_log2;
        next_finite = own < INF;
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full(t));
    };
    if (warp < TILES) {
        walk([&](const Item& it) {
            const uint32_t n = it.n;
            const int blocks = it.blocks, t = warp;
            if (threadIdx.x == 0 && (it.j0 != 0 || it.j1 != c.units)) { split[it.j0 == 0 ? 1 : 0] = c; is_split[it.j0 == 0 ? 1 : 0] = 1; }
            __syncwarp();
            if (elect_one()) {
                if (t < it.tiles) {
                    constexpr uint32_t HI = smem_desc_hi_sw128(1024);
                    const uint32_t q_lo = smem_desc_lo(sQ + t * SM::Q_BYTES, 16), k_lo0 = smem_desc_lo(sK, 16), v_lo0 = smem_desc_lo(sV, KV_SLAB);
                    const uint32_t cols = tmem_base + t * TILE_COLS;
                    auto issue_qk = [&](uint32_t b, uint32_t s) {            // S[s&1] = Q K_b^T
                        const uint32_t k_lo = k_lo0 + (b & 1) * (SM::KV_TILE >> 4);
#pragma unroll
                        for (int ks = 0; ks < D / 16; ++ks)
                            umma_f16(cols + (s & 1) * BK, smem_desc_join(q_lo + (((ks / 4) * Q_SLAB + (ks % 4) * 32) >> 4), HI),
                                     smem_desc_join(k_lo + (((ks / 4) * KV_SLAB + (ks % 4) * 32) >> 4), HI), IDESC_QK, ks != 0);
                        umma_commit(s_full(t, s & 1));
                        umma_commit(k_empty + 8 * (b & 1));
                    };
                    ok = mbar_wait(q_full(t), done & 1, p.status, 0x63);
                    for (int i = 0; i < 2 && i < blocks && ok; ++i) {        // two score blocks in flight before the first P arrives
                        const uint32_t b = n + i;
                        ok = mbar_wait(k_full + 8 * (b & 1), (b >> 1) & 1, p.status, 0x64);
                        tc_fence_after();
                        if (ok) issue_qk(b, pv + i);
                    }
                    for (int i = 0; i < blocks && ok; ++i) {
                        const uint32_t b = n + i, st = b & 1, par = (b >> 1) & 1, s = pv + i, v_lo = v_lo0 + st * (SM::KV_TILE >> 4);
                        ok = mbar_wait(v_full + 8 * st, par, p.status, 0x65) && mbar_wait(p_full(t, s & 1), (s >> 1) & 1, p.status, 0x66);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (int ks = 0; ks < BK / 16; ++ks)
                            umma_f16_ts(cols + O_COL, cols + (s & 1) * BK + ks * 8, smem_desc_join(v_lo + ks * (2048 >> 4), HI), IDESC_PV, (i | ks) != 0 ? 1u : 0u);
                        umma_commit(pv_done(t));
                        umma_commit(v_empty + 8 * st);
                        if (i + 1 == blocks) umma_commit(o_done(t));
                        if (i + 2 < blocks) {                                // S[s & 1] is free once this P V is in the pipe ahead
                            ok = mbar_wait(k_full + 8 * st, ((b + 2) >> 1) & 1, p.status, 0x67);
                            tc_fence_after();
                            if (ok) issue_qk(b + 2, s + 2);
                        }
                    }
                } else {
                    for (uint32_t b = n; b < n + blocks && ok; ++b) {        // no rows for this tile: it has no use for the operands
                        ok = mbar_wait(k_full + 8 * (b & 1), (b >> 1) & 1, p.status, 0x6f);
                        if (ok) mbar_arrive(k_empty + 8 * (b & 1));
                        ok = ok && mbar_wait(v_full + 8 * (b & 1), (b >> 1) & 1, p.status, 0x6f);
                        if (ok) mbar_arrive(v_empty + 8 * (b & 1));
                    }
                }
            }
            ok = __all_sync(0xffffffffu, ok);
            if (t < it.tiles) { pv += blocks; ++done; }
        });
    } else if (warp == COPY_WARP) {
        walk([&](const Item& it) {
            const uint32_t items = it.number, n = it.n;
            const int j0 = it.j0, j1 = it.j1, kend = it.kend;
            // Lane 4 x + g holds block and scales of 16-token group g of unit base + x; lane 0 issues the copies, of as many tokens at a
            // time as lie in one block.
            if (lane == 0) left_out[items % RING] = 0;
            const int* table = p.table + static_cast<size_t>(c.r) * p.max_blocks;
            const int step = min(p.block_size, BK) / 16;                     // groups per copy
            auto block_of = [&](int j) {
                const int unit = j + (lane >> 2), key = unit * BK + (lane & 3) * 16;
                const int id = unit < j1 && key < kend ? __ldg(table + (key >> p.shift)) : -1;
                return static_cast<unsigned>(id) < static_cast<unsigned>(p.num_blocks) ? id : -1;
            };
            int id_next = block_of(j0);
            for (int j = j0; j < j1 && ok; j += 8) {
                const int id = id_next;
                id_next = block_of(j + 8);
                float ks = 0.0f, vs = 1.0f;
                if (id >= 0) {
                    const size_t at = static_cast<size_t>(id) * p.kv_heads + c.h;
                    ks = paged_clamp_scale(__ldg(p.k_scale + at)); vs = paged_clamp_scale(__ldg(p.v_scale + at));
                }
                const float4 about = make_float4(ks, log2f(vs), 1.0f / vs, 0.0f);
                for (int x = 0; x < 8 && j + x < j1; ++x) {
                    const uint32_t b = n + (j + x - j0), st = b % RAW;
                    ok = __all_sync(0xffffffffu, mbar_wait(raw_empty + 8 * st, ((b / RAW) & 1) ^ 1, p.status, 0x68));
                    if (!ok) break;
                    if ((lane >> 2) == x) info[(b % RING) * 4 + (lane & 3)] = about;
                    __syncwarp();
                    uint32_t bytes = 0;
                    for (int g = 0; g < 4; g += step) {
                        const int mine = __shfl_sync(0xffffffffu, id, x * 4 + g);
                        if (mine >= 0) bytes += step * 16 * D * 2;
                    }
                    if (lane == 0) mbar_arrive_expect_tx(raw_full + 8 * st, bytes);
                    for (int g = 0; g < 4; g += step) {
                        const int mine = __shfl_sync(0xffffffffu, id, x * 4 + g);
                        if (mine >= 0 && lane == 0) {
                            const int key = (j + x) * BK + g * 16;
                            const size_t at = ((static_cast<size_t>(mine) * p.kv_heads + c.h) * p.block_size + (key & (p.block_size - 1))) * D;
                            const uint32_t dst = sR + st * 2 * SM::RAW_TILE + g * 16 * D;
                            bulk_copy(dst, k_cache + at, step * 16 * D, raw_full + 8 * st);
                            bulk_copy(dst + SM::RAW_TILE, v_cache + at, step * 16 * D, raw_full + 8 * st);
                        }
                    }
                    __syncwarp();
                }
            }
        });
    } else if (warp >= CONVERT_WARP && warp < SOFTMAX_WARP) {
        walk([&](const Item& it) {
            const uint32_t items = it.number, n = it.n;
            const int j0 = it.j0, j1 = it.j1, kend = it.kend, all_see = it.all_see;
            // ---- codes to f16 operands.  Chunk x of a block: 16 codes of token x / (D / 16), from column 16 * (x % (D / 16)).
            constexpr int PER_ROW = D / 16, LOADS = BK * PER_ROW / CONVERTERS;
            const int ct = threadIdx.x - CONVERT_WARP * 32;
            auto convert = [&](uint32_t tile, const uint4 (&from)[LOADS]) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const int x = ct + i * CONVERTERS, t = x / PER_ROW, col = (x % PER_ROW) * 2;      // in 16-byte chunks of 8 f16
                    uint32_t h[8];
                    e4m3x4_to_f16x4(from[i].x, h[0], h[1]); e4m3x4_to_f16x4(from[i].y, h[2], h[3]);
                    e4m3x4_to_f16x4(from[i].z, h[4], h[5]); e4m3x4_to_f16x4(from[i].w, h[6], h[7]);
                    // eight threads write one token's line in both 64-column slabs, which lie on the same banks: those of the second slab
                    // write their odd chunk first
                    const uint32_t line = tile + (col >> 3) * KV_SLAB + t * 128, sw = t & 7, odd = (col >> 3) & 1;
                    const uint32_t first = ((col & 7) + odd) ^ sw, second = first ^ 1;
                    sts128(line + (first << 4), odd ? h[4] : h[0], odd ? h[5] : h[1], odd ? h[6] : h[2], odd ? h[7] : h[3]);
                    sts128(line + (second << 4), odd ? h[0] : h[4], odd ? h[1] : h[5], odd ? h[2] : h[6], odd ? h[3] : h[7]);
                }
            };
            // Tokens behind the last key and blocks outside the pool: whatever lies there becomes zero.
            auto none = [&](int j, int i, const float4 (&in)[4]) {
                const int x = (ct + i * CONVERTERS) / PER_ROW;
                return j * BK + x >= kend || (x < 16 ? in[0].x : x < 32 ? in[1].x : x < 48 ? in[2].x : in[3].x) == 0.0f;
            };
            auto about = [&](uint32_t b, float4 (&in)[4]) {
#pragma unroll
                for (int g = 0; g < 4; ++g) in[g] = info[(b % RING) * 4 + g];
                return in[0].x == 0.0f || in[1].x == 0.0f || in[2].x == 0.0f || in[3].x == 0.0f;
            };
            auto keys = [&](int j) {
                const uint32_t b = n + (j - j0), st = b & 1, raw = sR + (b % RAW) * 2 * SM::RAW_TILE;
                if (!__all_sync(0xffffffffu, mbar_wait(raw_full + 8 * (b % RAW), (b / RAW) & 1, p.status, 0x69))) return false;
                uint4 x[LOADS];
#pragma unroll
                for (int i = 0; i < LOADS; ++i) x[i] = lds128(raw + (ct + i * CONVERTERS) * 16);
                float4 in[4];
                if (about(b, in) || (j + 1) * BK > kend) {
#pragma unroll
                    for (int i = 0; i < LOADS; ++i) if (none(j, i, in)) x[i] = make_uint4(0, 0, 0, 0);
                }
                if (!__all_sync(0xffffffffu, mbar_wait(k_empty + 8 * st, ((b >> 1) & 1) ^ 1, p.status, 0x6a))) return false;
                convert(sK + st * SM::KV_TILE, x);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(k_full + 8 * st);
                return true;
            };
            auto values = [&](int j) {                                       // of a block whose keys this warp has converted
                const uint32_t b = n + (j - j0), st = b & 1, raw = sR + (b % RAW) * 2 * SM::RAW_TILE;
                uint4 x[LOADS];
#pragma unroll
                for (int i = 0; i < LOADS; ++i) x[i] = lds128(raw + SM::RAW_TILE + (ct + i * CONVERTERS) * 16);
                const bool cut = (j + 1) * BK > all_see;
                float4 in[4];
                if (about(b, in) || cut) {
                    // NaN values that some row does not see become zero too (0 * NaN would reach it)
                    bool nan = false;
#pragma unroll
                    for (int i = 0; i < LOADS; ++i) {
                        const bool zero = none(j, i, in);
                        uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            if (zero) w[y] = 0;
                            const uint32_t z = cut ? nan_bytes(w[y]) : 0u;
                            nan |= z != 0;
                            w[y] &= ~((z >> 7) * 0xffu);
                        }
                        x[i] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    if (nan) left_out[items % RING] = 1;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(raw_empty + 8 * (b % RAW));
                if (!__all_sync(0xffffffffu, mbar_wait(v_empty + 8 * st, ((b >> 1) & 1) ^ 1, p.status, 0x6b))) return false;
                convert(sV + st * SM::KV_TILE, x);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(v_full + 8 * st);
                return true;
            };
            // a block's keys before the values of the one before it: the products with them come first, and their buffer is free earlier
            ok = keys(j0);
            for (int j = j0; j < j1 && ok; ++j) {
                if (j + 1 < j1) ok = keys(j + 1);
                if (ok) ok = values(j);
            }
        });
    } else if (warp >= SOFTMAX_WARP) {
        queries(c);
        walk([&](const Item& it) {
            const uint32_t items = it.number, n = it.n;
            const int j0 = it.j0, j1 = it.j1, blocks = it.blocks, row0 = it.row0, rows = it.rows, all_see = it.all_see;
            const bool mine = t < it.tiles;
            const int row = t * BQ + in_tile, lim = paged_limit(p, c.q, (row0 + min(row, rows - 1)) / p.group);
            const float qs = next_qs;
            const bool finite = next_finite;
            float m = -INFINITY, l = 0.0f;
            const int warp_sees = __shfl_sync(0xffffffffu, lim, 0);          // keys that every row of the warp sees
            for (int i = 0; i < blocks && mine && ok; ++i) {
                const uint32_t b = n + i, s = pv + i, s_addr = lane_addr + (s & 1) * BK;
                ok = __all_sync(0xffffffffu, mbar_wait(s_full(t, s & 1), (s >> 1) & 1, p.status, 0x6c));
                if (!ok) break;
                tc_fence_after();
                const int k0 = (j0 + i) * BK;
                uint32_t r[64];
                tmem_ld_32x32(s_addr, reinterpret_cast<uint32_t (&)[32]>(r[0]));
                tmem_ld_32x32(s_addr + 32, reinterpret_cast<uint32_t (&)[32]>(r[32]));
                float4 in[4];
#pragma unroll
                for (int g = 0; g < 4; ++g) in[g] = info[(b % RING) * 4 + g];
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
                    ok = __all_sync(0xffffffffu, mbar_wait(pv_done(t), (s - 1) & 1, p.status, 0x6d));
                    if (!ok) break;
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
                if (lane == 0) mbar_arrive(p_full(t, s & 1));
            }
            // The next item's queries, before this one's result: its first products run meanwhile.  The last products with this tile's
            // present operand are over, for their scores have been read.
            if (ok) {
                PagedCursor next = c;
                if (paged_next<ROWS, BK>(p, next)) queries(next);
            }
            // the last P V has a barrier of its own, one completion per item: this warp may come to it when any number have completed
            if (mine && ok) ok = __all_sync(0xffffffffu, mbar_wait(o_done(t), done & 1, p.status, 0x6e));
            if (mine && ok) {
                tc_fence_after();
                const bool whole = j0 == 0 && j1 == c.units;
                float* part = p.partials + (static_cast<size_t>(blockIdx.x) * 2 + (j0 == 0 ? 1 : 0)) * (static_cast<size_t>(ROWS) * (D + 2));
                const float ref = m == -INFINITY ? 0.0f : m;
                if (!finite && l > 0.0f) l = __int_as_float(0x7fffffff);
                // Results leave in 64 contiguous bytes per row: through 2 KB of shared memory, 16-byte pieces XORed with the row, a thread
                // writes piece lane % 4 of rows lane / 4, lane / 4 + 8, ..
                const int at_row = row0 + min(row, rows - 1), token = at_row / p.group, head = c.h * p.group + (at_row - token * p.group);
                const size_t row_at = (static_cast<size_t>(c.q.start) + token) * p.out_stride + static_cast<size_t>(head) * D;
                T* to[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) to[y] = static_cast<T*>(p.out) + __shfl_sync(0xffffffffu, row_at, y * 8 + (lane >> 2)) + (lane & 3) * 8;
                const uint32_t pad = smem_u32(smem + SM::OUT_OFF) + (warp - SOFTMAX_WARP) * 2048;
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                // columns of NaN values that were left out and that this row sees
                uint32_t nan_cols[D / 32];
#pragma unroll
                for (int x = 0; x < D / 32; ++x) nan_cols[x] = 0;
                if (*reinterpret_cast<volatile int*>(left_out + items % RING)) {
                    for (int key = max(j0, all_see / BK) * BK; key < min(lim, j1 * BK); ++key) {
                        const int id = __ldg(p.table + static_cast<size_t>(c.r) * p.max_blocks + (key >> p.shift));
                        if (static_cast<unsigned>(id) >= static_cast<unsigned>(p.num_blocks)) continue;
                        const uint32_t* v = reinterpret_cast<const uint32_t*>(v_cache + ((static_cast<size_t>(id) * p.kv_heads + c.h) * p.block_size + (key & (p.block_size - 1))) * D);
#pragma unroll
                        for (int y = 0; y < D / 4; ++y) {
                            const uint32_t z = nan_bytes(__ldg(v + y)) >> 7;
                            nan_cols[y / 8] |= ((z & 1u) | ((z >> 7) & 2u) | ((z >> 14) & 4u) | ((z >> 21) & 8u)) << (4 * (y % 8));
                        }
                    }
                }
#pragma unroll
                for (int x = 0; x < D / 32; ++x) {
                    uint32_t r[32];
                    tmem_ld_32x32(lane_addr + O_COL + x * 32, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int y = 0; y < 32; y += 8) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            v[e] = l == 0.0f ? 0.0f : __uint_as_float(r[y + e]);          // no key seen: whatever the products left
                            if (nan_cols[x] >> (y + e) & 1u) v[e] = __int_as_float(0x7fffffff);
                        }
                        if (whole) sts128(pad + lane * 64 + (((y >> 3) ^ ((lane >> 1) & 3)) << 4), paged_pack2<T>(v[0] * inv, v[1] * inv), paged_pack2<T>(v[2] * inv, v[3] * inv), paged_pack2<T>(v[4] * inv, v[5] * inv), paged_pack2<T>(v[6] * inv, v[7] * inv));
                        else if (row < rows) {
                            float4* dst = reinterpret_cast<float4*>(part) + (x * 8 + y / 4) * ROWS + row;
                            __stcg(dst, make_float4(v[0], v[1], v[2], v[3]));
                            __stcg(dst + ROWS, make_float4(v[4], v[5], v[6], v[7]));
                        }
                    }
                    __syncwarp();
                    if (whole) {
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            const int rr = y * 8 + (lane >> 2);
                            if (row - lane + rr < rows) *reinterpret_cast<uint4*>(to[y] + x * 32) = lds128(pad + rr * 64 + (((lane & 3) ^ ((rr >> 1) & 3)) << 4));
                        }
                    }
                    __syncwarp();
                }
                if (whole && row < rows && p.lse) p.lse[(static_cast<size_t>(c.q.start) + token) * (static_cast<size_t>(p.group) * p.kv_heads) + head] = l == 0.0f ? -INFINITY : (ref + log2f(l)) * 0.69314718055994531f;
                if (!whole && row < rows) { __stcg(part + ROWS * D + row, m); __stcg(part + ROWS * (D + 1) + row, l); }
                tc_fence_before();
                __syncwarp();
            }
            if (mine) { pv += blocks; ++done; }
        });
    }
    tc_fence_before();
    __syncthreads();
    if (*reinterpret_cast<volatile int*>(p.status) != ST_OK) for (int i = 0; i < 2000; ++i) __nanosleep(1000);       // let what is in flight land
    tc_fence_after();
    if (warp == 0) tmem_dealloc(tmem_base, TMEM_COLS);
    paged_announce<T, D, THREADS, ROWS>(p, shares, split, is_split, flags);
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

int paged_chunk_ctas() { return std::min(sm_count(), 320); }
size_t paged_chunk_partial_bytes(int head_dim) { return static_cast<size_t>(paged_chunk_ctas()) * 2 * ROWS * (head_dim + 2) * sizeof(float); }

int launch_paged_chunk(pyc_dtype dtype, int head_dim, PagedParams p, const void* k_cache, const void* v_cache, cudaStream_t s) {
    // an item's queries, first blocks and result weigh as much as this many units of 64 keys: 3 373 us, 6 357, 10 346, 14 348, 20 357 for
    // 2048-query chunks; 8 prompts of 1000 tokens 223, 192, 176, 183, 183
    p.cost = 10; p.unsplit = 16;
    if (dtype == PYC_DTYPE_F16) return head_dim == 128 ? launch<__half, 128>(p, k_cache, v_cache, s) : launch<__half, 64>(p, k_cache, v_cache, s);
    return head_dim == 128 ? launch<__nv_bfloat16, 128>(p, k_cache, v_cache, s) : launch<__nv_bfloat16, 64>(p, k_cache, v_cache, s);
}

}  // namespace b200
