// Attention of a ragged batch of queries over the 8-bit paged key/value cache (layout and meaning: include/pyc_b200.h).
// PyC has no counterpart; the dense kernels are in attention.cu.
//
// This file: few query rows per key head (single new tokens, a few of them, grouped heads), which is bound by reading the
// cache.  A CTA walks the items of its stretch (paged_attention.cuh).  Each of its warps takes 32 keys of every unit
// and runs on its own: its own ring of TMA copies (keys and values, one copy each or two where a block is 16 tokens, into
// 128-byte swizzled shared memory), its own running maximum and sums in registers, no barrier with the other warps before
// the item's end.  At an item's end the next item's first copies are asked for before the warps' sums are joined, and split
// items are announced at the end of the stretch: an item's end costs 5 to 9 us of waiting for ids, scales, queries, fences
// and counters, which passes beside the copies that way.  Measured: 64 requests of up to 8000 keys (8 x 4 heads of 128, blocks of 16,
// bf16, 584 MB of cache) 105 us = 5.6 TB/s, 0.85 of the measured copy rate; one of 131085 keys (269 MB, f16) 60 us = 4.5 TB/s, of which
// the beginning of the shares takes about 5 us and the join as many.
//
// Products, on the warp-level tensor instructions (an item has 1 to 32 rows; a 128-row tcgen05 tile would be empty), both
// transposed so that keys and head dimension fill the instruction's 16 rows and 8 queries its columns:
//   S^T = K Q^T  m16n8k32 e4m3 x e4m3 -> f32.  The keys' codes are the operand as they lie in the cache, nothing is converted;
//                the queries are split into e4m3 terms.  (As an f16 product with converted keys, a third of all
//                instructions were conversions.)
//   O^T = V^T P^T  m16n8k16 f16.  The values' codes become f16 exactly, two per conversion; P^T comes from the score
//                fragment by an 8 x 8 transpose between lanes.
// Which head_dim value sits at which position of a contraction is free as long as both operands agree, and so is the order
// of the result's rows: thread (g = lane / 4, c = lane % 4) takes the D / 4 consecutive values from c * D / 4 of keys g, g + 8, ..,
// and the D / 8 consecutive values from g * D / 8 of keys 2c, 2c + 1, 2c + 8, ...  So 16-byte shared-memory loads,
// conflict-free under the swizzle, feed the tensor cores.
//
// Precision.  A query row is scaled by a power of two to [128, 256) and split: e4m3(q), then 16 times the rest, once for
// bf16 and twice for f16; 4 + 4 (+ 4) significant bits hold the type's 8 (11) exactly, but for values below 2^-13 of the
// row's largest, which keep an absolute error of 2^-21 of it.  The products are exact and added in f32.
// The value scale vs of a block joins the exponent, p' = 2^(score + log2 vs - m), with m the running maximum of score +
// log2 vs, so the f16 operand holds the weight with which the block's CODES enter the sum: its largest is near 1 whatever the
// scales, and f16's 11 bits hold (2^-12 relative error, 2^-25 absolute below 2^-14).  The softmax's weight is sum p' / vs in
// f32.  m only moves when a score exceeds it by more than 2^8 (p' stays far below f16's 65504): a vote of the warp finds
// that out, and only then the maximum is formed across lanes and the sums are rescaled.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "internal.h"
#include "paged_attention.cuh"
#include "paged_attention_chunk.h"
#include "ptx_sm100.cuh"

namespace b200 {
namespace {

constexpr int GROUP = 32;                    // keys that a warp takes at a time

// NQ: 8-row query tiles per item.
template <int D, int NQ>
struct ShortCfg {
    static constexpr int ROWS = NQ * 8;                                    // query rows per item
    static constexpr int NW = NQ <= 2 ? 4 : 8;                             // warps per CTA
    static constexpr int PER_SM = NQ == 1 ? 3 : NQ == 2 ? 2 : 1;           // resident CTAs
    static constexpr int THREADS = NW * 32;
    static constexpr int UNIT = NW * GROUP;                                // keys per unit
    static constexpr int TILE = GROUP * D;                                 // bytes of a group's keys (or values)
    static constexpr int RING_BYTES = (NQ == 1 ? 64 : NQ == 2 ? 96 : 192) * 1024;
    static constexpr int STAGES = RING_BYTES / (NW * 2 * TILE);
    static constexpr int TERM_BYTES = ROWS * D;                            // one e4m3 term of the queries, in operand order
    static constexpr int Q_OFF = RING_BYTES;
    static constexpr int ROW_OFF = Q_OFF + 3 * TERM_BYTES;                // float [ROWS] row scales
    static constexpr int ML_OFF = ROW_OFF + ROWS * 4;                      // float [NW][ROWS][2]
    static constexpr int INFO_OFF = ML_OFF + NW * ROWS * 8;                // float4 [NW][STAGES][2]
    static constexpr int BAR_OFF = INFO_OFF + NW * STAGES * 32;            // mbarriers [NW][STAGES]
    static constexpr int SHARES_OFF = BAR_OFF + NW * STAGES * 8;
    static constexpr int SPLIT_OFF = SHARES_OFF + sizeof(PagedShares);     // PagedCursor [2], int [2], int [2]
    static constexpr int BYTES = SPLIT_OFF + 2 * sizeof(PagedCursor) + 16;
    static constexpr int EARLY = NQ <= 2 ? 1 : 0;                          // groups of the next item that are asked for before this one's sums are joined
    static_assert(ROWS * D * 4 <= (EARLY ? 1 : STAGES) * 2 * TILE, "a warp's sums beside them");
    static_assert(SHARES_OFF % 8 == 0 && STAGES >= 2 && STAGES <= 16 && (BYTES + 1024) * PER_SM <= 228 * 1024, "shared memory of an SM");
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 x 8 matrix of 16-bit values, two per lane (row lane / 4, columns 2c, 2c + 1), transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
// Byte `o` of a tile that TMA wrote with the 128-byte swizzle (16-byte chunks of each 128-byte line XORed with the line's number mod 8).
__device__ __forceinline__ uint32_t swizzled(uint32_t o) { return o ^ ((o >> 3) & 0x70u); }
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }
// 0x80 in each byte that is a NaN code.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

template <typename T, int D, int NQ>
__global__ void __launch_bounds__(ShortCfg<D, NQ>::THREADS, ShortCfg<D, NQ>::PER_SM)
paged_short_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PagedParams p, int halves) {
    using SM = ShortCfg<D, NQ>;
    constexpr int NW = SM::NW, THREADS = SM::THREADS, UNIT = SM::UNIT;
    constexpr int TILE = SM::ROWS, S = SM::STAGES, KC = D / 64, NT = D / 8;  // KC: 16-byte chunks of a key per thread; NT: values of a token per thread
    constexpr int TERMS = std::is_same<T, __half>::value ? 3 : 2;
    extern __shared__ __align__(1024) uint8_t smem[];                        // the swizzle goes by address bits: the copies' memory starts on 1024 bytes
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c4 = lane & 3;
    float* row_scale = reinterpret_cast<float*>(smem + SM::ROW_OFF);
    float* warp_ml = reinterpret_cast<float*>(smem + SM::ML_OFF);
    PagedShares& shares = *reinterpret_cast<PagedShares*>(smem + SM::SHARES_OFF);
    PagedCursor (&split)[2] = *reinterpret_cast<PagedCursor (*)[2]>(smem + SM::SPLIT_OFF);
    int (&is_split)[2] = *reinterpret_cast<int (*)[2]>(smem + SM::SPLIT_OFF + 2 * sizeof(PagedCursor));
    int* flags = reinterpret_cast<int*>(smem + SM::SPLIT_OFF + 2 * sizeof(PagedCursor) + 8);
    float4* info = reinterpret_cast<float4*>(smem + SM::INFO_OFF) + w * S * 2;
    const uint32_t bars = smem_u32(smem + SM::BAR_OFF) + w * S * 8;
    const uint32_t ring = smem_u32(smem) + w * S * 2 * SM::TILE;
    const uint32_t q_frags = smem_u32(smem + SM::Q_OFF) + lane * 16;         // [term][query tile][64 values of D][lane]: 16 bytes

    if (lane == 0) {
        for (int i = 0; i < S; ++i) mbar_init(bars + 8 * i, halves);
        fence_barrier_init();
        fence_proxy_async();
        if (w == 0) is_split[0] = is_split[1] = 0;
    }
    PagedCursor c;
    const bool busy = paged_begin<THREADS, TILE, UNIT>(p, c, shares);
    __syncthreads();
    if (!busy) return;
    bool ok = true;

    // ---- the warp's copies.  A group lies in one block (halves = 1, block sizes from 32) or in two of 16 tokens (halves = 2).  Lane
    // unit * halves + half, counted from unit `base`, has the id and scales of one of them and issues its copies.
    const int mine_u = halves == 2 ? lane >> 1 : lane, mine_h = halves == 2 ? lane & 1 : 0;
    int base = 0, id = -1;                   // block (-1: masked)
    float ks = 0.0f, vs = 1.0f;              // its scales as loaded
    float4 about;                            // key scale (0: masked), log2 of the value scale, 1 / it
    auto block_of = [&](const PagedCursor& at, int j, int j1, int kend) {    // asked for; the caller checks its range
        const int key = (j + mine_u) * UNIT + w * GROUP + mine_h * 16;
        return j + mine_u < j1 && key < kend ? __ldg(p.table + static_cast<size_t>(at.r) * p.max_blocks + (key >> p.shift)) : -1;
    };
    auto take = [&](int j, int block) { base = j; id = static_cast<unsigned>(block) < static_cast<unsigned>(p.num_blocks) ? block : -1; };
    auto scales = [&]() {                    // asked for; `describe` waits for them
        ks = 0.0f; vs = 1.0f;
        if (id >= 0) {
            const size_t at = static_cast<size_t>(id) * p.kv_heads + c.h;
            ks = __ldg(p.k_scale + at); vs = __ldg(p.v_scale + at);
        }
    };
    auto describe = [&]() {
        vs = paged_clamp_scale(vs);
        about = make_float4(id >= 0 ? paged_clamp_scale(ks) : 0.0f, log2f(vs), 1.0f / vs, 0.0f);
    };
    auto copy = [&](int j, uint32_t at) {    // unit j's group into stage `at`; all lanes call it
        if (mine_u == j - base) {
            if (id >= 0) {
                const uint32_t bytes = SM::TILE / halves, dst = ring + at * 2 * SM::TILE + mine_h * (SM::TILE / 2);
                const int y = ((j * UNIT + w * GROUP + mine_h * 16) & (p.block_size - 1)) * D / 128, z = id * p.kv_heads + c.h;
                mbar_arrive_expect_tx(bars + 8 * at, 2 * bytes);
                tma_load_3d(dst, &tmK, bars + 8 * at, 0, y, z);
                tma_load_3d(dst + SM::TILE, &tmV, bars + 8 * at, 0, y, z);
            } else mbar_arrive(bars + 8 * at);
        }
    };
    auto note = [&](int j, uint32_t at) {    // what the products have to know about it
        if (mine_u == j - base) {
            info[at * 2 + mine_h] = about;
            if (halves == 1) info[at * 2 + 1] = about;
        }
    };
    uint32_t st = 0, parity = 0;             // stage that is read next, parity of its completion
    auto stage = [&](int i) { const uint32_t at = st + i; return at >= S ? at - S : at; };   // i < S stages on
    // ---- the queries: 16 threads per row, D / 16 values each; loaded an item ahead
    constexpr int PARTS = (TILE * 16 + THREADS - 1) / THREADS, NV = D / 16;
    uint32_t q_raw[PARTS][NV / 2];
    auto load_q = [&](const PagedCursor& at) {
        const int row0 = at.t * TILE, rows = min(TILE, at.q.rows - row0);
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            const int row = part * (THREADS / 16) + (threadIdx.x >> 4), x = threadIdx.x & 15;
#pragma unroll
            for (int i = 0; i < NV / 2; ++i) q_raw[part][i] = 0;
            if (row < rows) {
                const int token = (row0 + row) / p.group, head = at.h * p.group + (row0 + row - token * p.group);
                const T* src = static_cast<const T*>(p.q) + (static_cast<size_t>(at.q.start) + token) * p.q_stride + static_cast<size_t>(head) * D + x * NV;
                if constexpr (NV == 8) { const uint4 v = __ldg(reinterpret_cast<const uint4*>(src)); q_raw[part][0] = v.x; q_raw[part][1] = v.y; q_raw[part][2] = v.z; q_raw[part][3] = v.w; }
                else { const uint2 v = __ldg(reinterpret_cast<const uint2*>(src)); q_raw[part][0] = v.x; q_raw[part][1] = v.y; }
            }
        }
    };

    int ahead;                               // block of the next item's first groups
    {
        const int j0 = c.from(), j1 = c.to();
        take(j0, block_of(c, j0, j1, paged_tile_end<TILE>(p, c.q, c.t)));
        load_q(c);
#pragma unroll 1
        for (int i = 0; i < S && j0 + i < j1; ++i) copy(j0 + i, i);
        scales();
    }

    // this thread's places in a stage: keys g (+ 8, 16, 24) and values 2c, 2c + 1 (+ 8, ...).  8 lines on the swizzle repeats: that
    // is 8 keys for D = 128 and 16 for D = 64, where 8 keys on the chunk's bit 2 (64 bytes) is the other one
    constexpr int ODD = D == 64 ? 64 : 0;
    uint32_t k_at[KC][2], v_at[2][2];
#pragma unroll
    for (int i = 0; i < KC; ++i) { k_at[i][0] = swizzled(g * D + c4 * (D / 4) + i * 16); k_at[i][1] = k_at[i][0] ^ ODD; }
#pragma unroll
    for (int i = 0; i < 2; ++i) { v_at[i][0] = swizzled((2 * c4 + i) * D + g * NT); v_at[i][1] = v_at[i][0] ^ ODD; }

    for (;;) {
        const int j0 = c.from(), j1 = c.to();
        const int row0 = c.t * TILE, rows = min(TILE, c.q.rows - row0);
        const int kend = paged_tile_end<TILE>(p, c.q, c.t);

        // ---- queries to e4m3 terms in operand order
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            const int row = part * (THREADS / 16) + (threadIdx.x >> 4), x = threadIdx.x & 15;
            float v[NV];
            float amax = 0.0f;
            bool finite = true;
#pragma unroll
            for (int i = 0; i < NV / 2; ++i) {
                const float2 f = unpack2<T>(q_raw[part][i]);
                v[2 * i] = f.x; v[2 * i + 1] = f.y;
                amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
                finite &= fabsf(f.x) < INFINITY && fabsf(f.y) < INFINITY;
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o, 16));
            const unsigned all = __ballot_sync(0xffffffffu, finite);
            const bool row_finite = ((all >> (lane & 16)) & 0xffffu) == 0xffffu;
            // 2^-e brings the largest to [128, 256) (below 2^-119, where 2^-e leaves the range, to less)
            const int e = amax > 0.0f && row_finite ? max(static_cast<int>(__float_as_uint(amax) >> 23) - 134, -126) : 0;
            const float down = exp2_int(-e);
            if (row < TILE) {
                if (x == 0) row_scale[row] = row_finite ? exp2_int(e) * p.scale_log2 : __int_as_float(0x7fffffff);
                float f[NV];
#pragma unroll
                for (int i = 0; i < NV; ++i) f[i] = row_finite ? v[i] * down : 0.0f;
                // operand position of values d .. d + 3 (d = 4 * word of thread c's D / 4): chunk of 16 values, then word
#pragma unroll
                for (int i = 0; i < NV; i += 4) {
                    const int d = x * NV + i, cc = d / (D / 4), word = (d % (D / 4)) / 4;
                    uint8_t* dst = smem + SM::Q_OFF + (((row >> 3) * KC + word / 4) * 32 + (row & 7) * 4 + cc) * 16 + (word & 3) * 4;
#pragma unroll
                    for (int term = 0; term < TERMS; ++term) {
                        const uint32_t q4 = e4m3x4(f[i], f[i + 1], f[i + 2], f[i + 3]);
                        *reinterpret_cast<uint32_t*>(dst + term * SM::TERM_BYTES) = q4;
                        const float2 lo = e4m3x2_to_float2(q4 & 0xffffu), hi = e4m3x2_to_float2(q4 >> 16);
                        const float up = term == 0 ? 16.0f : 1.0f;           // the rests share one scale and one accumulator
                        f[i] = (f[i] - lo.x) * up; f[i + 1] = (f[i + 1] - lo.y) * up; f[i + 2] = (f[i + 2] - hi.x) * up; f[i + 3] = (f[i + 3] - hi.y) * up;
                    }
                }
            }
        }
        describe();
#pragma unroll 1
        for (int i = 0; i < S && j0 + i < j1; ++i) note(j0 + i, stage(i));
        PagedCursor then = c;
        const bool more = paged_next<TILE, UNIT>(p, then);
        ahead = -1;
        if (more) {                          // what the next item begins with
            ahead = block_of(then, 0, then.to(), paged_tile_end<TILE>(p, then.q, then.t));
            load_q(then);
        }
        __syncthreads();

        // this thread's queries: 2c and 2c + 1 of every tile
        int lim[NQ][2];
        float qs[NQ][2];
#pragma unroll
        for (int t = 0; t < NQ; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = t * 8 + 2 * c4 + i;
                lim[t][i] = row < rows ? paged_limit(p, c.q, (row0 + row) / p.group) : kend;
                qs[t][i] = row_scale[row];
            }
        const int all_see = paged_limit(p, c.q, row0 / p.group);             // keys that every row sees

        float o[NQ][D / 16][4], m[NQ][2], l[NQ][2];                          // o: values g * NT + 2n (0, 1) and + 1 (2, 3) of the two queries
#pragma unroll
        for (int t = 0; t < NQ; ++t) {
#pragma unroll
            for (int i = 0; i < 2; ++i) { m[t][i] = -INFINITY; l[t][i] = 0.0f; }
#pragma unroll
            for (int n = 0; n < D / 16; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[t][n][i] = 0.0f;
        }

#pragma unroll 1
        for (int j = j0; j < j1; ++j) {
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bars + 8 * st, parity, p.status, 0x61));
            const float4 in0 = info[st * 2], in1 = info[st * 2 + 1];
            const uint32_t kt = ring + st * 2 * SM::TILE, vt = kt + SM::TILE;
            const int key0 = j * UNIT + w * GROUP;
            // scores of keys g, g + 8, g + 16, g + 24 with this thread's queries: s[tile][key group of 16][key 0/8, query 0/1]
            float s[NQ][2][4], r[NQ][2][4];
#pragma unroll
            for (int t = 0; t < NQ; ++t)
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) { s[t][k][i] = 0.0f; r[t][k][i] = 0.0f; }
#pragma unroll
            for (int i = 0; i < KC; ++i) {
                uint4 kk[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) kk[t] = lds128(kt + k_at[i][t & 1] + t * 8 * D);
#pragma unroll
                for (int t = 0; t < NQ; ++t)
#pragma unroll
                    for (int term = 0; term < TERMS; ++term) {
                        const uint4 q = lds128(q_frags + term * SM::TERM_BYTES + (t * KC + i) * 512);
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            float (&acc)[4] = term == 0 ? s[t][k] : r[t][k];
                            mma_e4m3(acc, kk[2 * k].x, kk[2 * k + 1].x, kk[2 * k].y, kk[2 * k + 1].y, q.x, q.y);
                            mma_e4m3(acc, kk[2 * k].z, kk[2 * k + 1].z, kk[2 * k].w, kk[2 * k + 1].w, q.z, q.w);
                        }
                    }
            }
            const bool cut = key0 + GROUP > all_see || in0.x == 0.0f || in1.x == 0.0f;          // some row does not see some key of the group
            uint32_t pb[NQ][4];                                              // P^T operands of 8 keys each
            bool above = false;
#pragma unroll
            for (int t = 0; t < NQ; ++t) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float f = qs[t][i & 1] * (k ? in1.x : in0.x);
                        s[t][k][i] = fmaf(fmaf(r[t][k][i], 0.0625f, s[t][k][i]), f, k ? in1.y : in0.y);
                    }
                if (cut) {
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if ((k ? in1.x : in0.x) == 0.0f || key0 + k * 16 + (i >> 1) * 8 + g >= lim[t][i & 1]) s[t][k][i] = -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) above |= fmaxf(fmaxf(s[t][0][i], s[t][0][2 + i]), fmaxf(s[t][1][i], s[t][1][2 + i])) > m[t][i] + 8.0f;   // also from -inf
            }
            if (__any_sync(0xffffffffu, above)) {
#pragma unroll
                for (int t = 0; t < NQ; ++t) {
                    float alpha[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float mx = fmaxf(fmaxf(s[t][0][i], s[t][0][2 + i]), fmaxf(s[t][1][i], s[t][1][2 + i]));
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                        const bool move = mx > m[t][i] + 8.0f;
                        alpha[i] = move ? ex2_approx(m[t][i] - mx) : 1.0f;
                        if (move) m[t][i] = mx;
                        l[t][i] *= alpha[i];
                    }
#pragma unroll
                    for (int n = 0; n < D / 16; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[t][n][i] *= alpha[i & 1];
                }
            }
#pragma unroll
            for (int t = 0; t < NQ; ++t) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float ref = m[t][i] == -INFINITY ? 0.0f : m[t][i];
#pragma unroll
                    for (int k = 0; k < 2; ++k) { s[t][k][i] = ex2_approx(s[t][k][i] - ref); s[t][k][2 + i] = ex2_approx(s[t][k][2 + i] - ref); }
                    l[t][i] = fmaf(s[t][0][i] + s[t][0][2 + i], in0.z, fmaf(s[t][1][i] + s[t][1][2 + i], in1.z, l[t][i]));
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const __half2 h = __floats2half2_rn(s[t][k >> 1][(k & 1) * 2], s[t][k >> 1][(k & 1) * 2 + 1]);
                    pb[t][k] = transpose8(*reinterpret_cast<const uint32_t*>(&h));
                }
            }
            // values, 16 keys at a time: keys 2c, 2c + 1, 2c + 8, 2c + 9, D / 8 codes each
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t v[4][NT / 4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t a = vt + v_at[i & 1][i >> 1] + (half * 16 + (i >> 1) * 8) * D;
                    if constexpr (NT == 16) { const uint4 x = lds128(a); v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w; }
                    else { const uint2 x = lds64(a); v[i][0] = x.x; v[i][1] = x.y; }
                }
                bool own_nan = false;
                if (cut) {
                    const bool gone = (half ? in1.x : in0.x) == 0.0f;
                    uint32_t nans = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool past = gone || key0 + half * 16 + 2 * c4 + (i & 1) + (i >> 1) * 8 >= kend;
#pragma unroll
                        for (int x = 0; x < NT / 4; ++x) {
                            if (past) v[i][x] = 0;                       // behind the last key of the tile: whatever is there
                            const uint32_t z = nan_codes(v[i][x]);
                            nans |= z;
                            v[i][x] &= ~((z >> 7) * 0xffu);              // 0 * NaN would reach the rows that do not see it
                        }
                    }
                    own_nan = __any_sync(0xffffffffu, nans != 0);
                }
#pragma unroll
                for (int x = 0; x < NT / 4; ++x) {
                    // bytes of two keys side by side: (key, key + 1) for values 4x, 4x + 1 | 4x + 2, 4x + 3
                    uint32_t a[4], b[4];
                    e4m3x4_to_f16x4(prmt(v[0][x], v[1][x], 0x5140), a[0], a[1]);
                    e4m3x4_to_f16x4(prmt(v[0][x], v[1][x], 0x7362), a[2], a[3]);
                    e4m3x4_to_f16x4(prmt(v[2][x], v[3][x], 0x5140), b[0], b[1]);
                    e4m3x4_to_f16x4(prmt(v[2][x], v[3][x], 0x7362), b[2], b[3]);
#pragma unroll
                    for (int t = 0; t < NQ; ++t) {
                        mma_f16(o[t][2 * x], a[0], a[1], b[0], b[1], pb[t][2 * half], pb[t][2 * half + 1]);
                        mma_f16(o[t][2 * x + 1], a[2], a[3], b[2], b[3], pb[t][2 * half], pb[t][2 * half + 1]);
                    }
                }
                if (own_nan) {                                           // NaN values in a group that not every row sees whole: only to the rows that see them
                    for (int k = 0; k < 16; ++k) {
                        const int key = key0 + half * 16 + k;
                        if (key >= kend) break;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            uint32_t byte;
                            asm volatile("ld.shared.u8 %0, [%1];" : "=r"(byte) : "r"(vt + swizzled((half * 16 + k) * D + g * NT + n)));
                            if ((byte & 127u) == 127u) {
#pragma unroll
                                for (int t = 0; t < NQ; ++t)
#pragma unroll
                                    for (int i = 0; i < 2; ++i)
                                        if (key < lim[t][i]) o[t][n >> 1][(n & 1) * 2 + i] = __int_as_float(0x7fffffff);
                            }
                        }
                    }
                }
            }
            __syncwarp();
            if (ok && j + S < j1) {
                if ((j + S - base) * halves >= 32) { take(j + S, block_of(c, j + S, j1, kend)); scales(); describe(); }
                copy(j + S, st);
                note(j + S, st);
            }
            __syncwarp();
            if (++st == S) { st = 0; parity ^= 1; }
        }

        // ---- the item's end: the next item's first groups, then the warps' sums, which meet in the memory of later groups
        const PagedCursor done = c;
        if (more) {
            paged_next<TILE, UNIT>(p, c);
            take(0, ahead);
            if (ok && SM::EARLY) copy(0, st);
            scales();
        }
        constexpr int SUM_STRIDE = S * 2 * SM::TILE / 4;                     // floats between two warps' rings
        float* sums = reinterpret_cast<float*>(smem) + (SM::EARLY ? stage(1) * (2 * SM::TILE / 4) : 0);
#pragma unroll
        for (int t = 0; t < NQ; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], x);
                const int row = t * 8 + 2 * c4 + i;
                if (row < rows) {
                    if (g == 0) { warp_ml[(w * TILE + row) * 2] = m[t][i]; warp_ml[(w * TILE + row) * 2 + 1] = l[t][i]; }
                    float* dst = sums + w * SUM_STRIDE + row * D + g * NT;
#pragma unroll
                    for (int n = 0; n < D / 16; n += 2)
                        *reinterpret_cast<float4*>(dst + 2 * n) = make_float4(o[t][n][i], o[t][n][2 + i], o[t][n + 1][i], o[t][n + 1][2 + i]);
                }
            }
        __syncthreads();
        const bool whole = j0 == 0 && j1 == done.units;
        float* part = p.partials + (static_cast<size_t>(blockIdx.x) * 2 + (j0 == 0 ? 1 : 0)) * (static_cast<size_t>(TILE) * (D + 2));
        for (int e = threadIdx.x; e < rows * (D / 4); e += THREADS) {
            const int row = e / (D / 4), d = (e % (D / 4)) * 4;
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < NW; ++i) mx = fmaxf(mx, warp_ml[(i * TILE + row) * 2]);
            const float ref = mx == -INFINITY ? 0.0f : mx;
            float sum = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                const float f = ex2_approx(warp_ml[(i * TILE + row) * 2] - ref);
                const float4 y = *reinterpret_cast<const float4*>(sums + i * SUM_STRIDE + row * D + d);
                sum = fmaf(warp_ml[(i * TILE + row) * 2 + 1], f, sum);
                v[0] = fmaf(y.x, f, v[0]); v[1] = fmaf(y.y, f, v[1]); v[2] = fmaf(y.z, f, v[2]); v[3] = fmaf(y.w, f, v[3]);
            }
            if (whole) paged_finish<T, D>(p, done, row0 + row, d, v, ref, sum);
            else {
                __stcg(reinterpret_cast<float4*>(part + row * D + d), make_float4(v[0], v[1], v[2], v[3]));
                if (d == 0) { __stcg(part + TILE * D + row, mx); __stcg(part + TILE * (D + 1) + row, sum); }
            }
        }
        if (!whole && threadIdx.x == 0) { split[j0 == 0 ? 1 : 0] = done; is_split[j0 == 0 ? 1 : 0] = 1; }
        if (!more) break;
        fence_proxy_async();                                                 // the sums' memory goes back to the copies
        __syncthreads();
        if (ok) {
#pragma unroll 1
            for (int i = SM::EARLY; i < S && i < c.to(); ++i) copy(i, stage(i));
        }
    }
    paged_announce<T, D, THREADS, TILE>(p, shares, split, is_split, flags);
    if (!ok) for (int i = 0; i < 2000; ++i) __nanosleep(1000);               // a wait has run out: let what is in flight land
}

template <typename T, int D, int NQ>
int launch_short(const CUtensorMap& tmK, const CUtensorMap& tmV, const PagedParams& p, int halves, cudaStream_t s) {
    using SM = ShortCfg<D, NQ>;
    auto kernel = paged_short_kernel<T, D, NQ>;
    B200_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::BYTES));
    kernel<<<sm_count() * SM::PER_SM, SM::THREADS, SM::BYTES, s>>>(tmK, tmV, p, halves);
    B200_CUDA_OK(cudaGetLastError());
    count_launch();
    return 0;
}

// Which kernel takes a request goes by its rows (queries times query heads of a key head).  Measured for 64 requests of 8000 keys,
// 8 key heads, bf16, this file's kernel | the tcgen05 kernel: head_dim 128, 8 rows 181 | 423 us, 16 rows 229 (f16 279) | 423, 32 rows
// 676 (spills) | 425; head_dim 64, 16 rows 169 | 384, 32 rows 292 | 385.
constexpr int few_rows(int head_dim) { return head_dim == 128 ? 16 : 32; }

constexpr size_t WS_COUNTERS = 4096;          // bytes: one int per CTA, at most 1024

// Two slots of [rows][D + 2] floats per CTA, for the largest of the forms.
size_t partial_bytes(int head_dim) {
    const int rows = std::max({ShortCfg<64, 1>::PER_SM * ShortCfg<64, 1>::ROWS, ShortCfg<64, 2>::PER_SM * ShortCfg<64, 2>::ROWS,
                               ShortCfg<64, 4>::PER_SM * ShortCfg<64, 4>::ROWS});
    return static_cast<size_t>(sm_count()) * rows * 2 * (head_dim + 2) * sizeof(float);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t pyc_b200_paged_attention_workspace_bytes(int requests, int max_query, int heads, int kv_heads, int head_dim) {
    if (requests < 1 || max_query < 1 || kv_heads < 1 || heads < kv_heads || heads % kv_heads || (head_dim != 64 && head_dim != 128)) return 0;
    const bool many = static_cast<long long>(max_query) * (heads / kv_heads) > few_rows(head_dim);
    return WS_COUNTERS + (many ? std::max(partial_bytes(head_dim), paged_chunk_partial_bytes(head_dim)) : partial_bytes(head_dim));
}

int pyc_b200_paged_attention(const pyc_b200_paged_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (!a || !a->q || !a->k_cache || !a->v_cache || !a->k_scale || !a->v_scale || !a->block_table || !a->query_start || !a->seq_lens || !a->out || !workspace) {
        set_error("paged attention: NULL argument"); return -1;
    }
    if (a->dtype != PYC_DTYPE_BF16 && a->dtype != PYC_DTYPE_F16) { set_error("paged attention: queries must be bf16 or f16"); return -1; }
    const int shift = kv_block_shift(a->block_size);
    if (shift < 0) { set_error("paged attention: block_size %d is not 16, 32, 64 or 128", a->block_size); return -1; }
    if (a->head_dim != 64 && a->head_dim != 128) { set_error("paged attention: head_dim %d is not 64 or 128", a->head_dim); return -1; }
    if (a->requests < 1 || a->requests > 16384 || a->max_query < 1 || a->num_blocks < 1 || a->max_blocks < 1) {
        set_error("paged attention: requests (1 .. 16384), max_query, num_blocks and max_blocks must be positive"); return -1;
    }
    if (a->rows < 0) { set_error("paged attention: %d rows", a->rows); return -1; }
    if (!(a->scale > 0.0f && a->scale < INFINITY)) { set_error("paged attention: scale must be positive and finite"); return -1; }
    if (a->kv_heads < 1 || a->heads < 1 || a->heads % a->kv_heads) { set_error("paged attention: %d heads over %d key heads", a->heads, a->kv_heads); return -1; }
    if (static_cast<long long>(a->num_blocks) * a->kv_heads > INT_MAX || static_cast<long long>(a->max_blocks) * a->block_size > INT_MAX ||
        static_cast<long long>(a->max_query) * (a->heads / a->kv_heads) > INT_MAX / 2) {
        set_error("paged attention: num_blocks * kv_heads, max_blocks * block_size or max_query * heads / kv_heads is too large"); return -1;
    }
    const size_t row = static_cast<size_t>(a->heads) * a->head_dim;
    const size_t qs = a->q_stride ? a->q_stride : row, os = a->out_stride ? a->out_stride : row;
    if (qs < row || os < row || qs % 8 || os % 8) { set_error("paged attention: row strides must be multiples of 8 and at least heads * head_dim"); return -1; }
    auto al = [](const void* x, size_t n) { return reinterpret_cast<uintptr_t>(x) % n == 0; };
    if (!al(a->q, 16) || !al(a->out, 16) || !al(a->k_cache, 16) || !al(a->v_cache, 16)) { set_error("paged attention: pointers must be 16-byte aligned"); return -1; }
    const size_t need = pyc_b200_paged_attention_workspace_bytes(a->requests, a->max_query, a->heads, a->kv_heads, a->head_dim);
    if (workspace_bytes < need) { set_error("paged attention: workspace of %zu bytes needed, %zu given", need, workspace_bytes); return -1; }
    if (!al(workspace, 256)) { set_error("paged attention: workspace must be 256-byte aligned"); return -1; }

    PagedParams p = {};
    p.q = a->q; p.out = a->out; p.lse = a->lse; p.k_scale = a->k_scale; p.v_scale = a->v_scale;
    p.table = a->block_table; p.starts = a->query_start; p.lens = a->seq_lens; p.q_stride = qs; p.out_stride = os;
    p.requests = a->requests; p.group = a->heads / a->kv_heads; p.kv_heads = a->kv_heads; p.max_query = a->max_query;
    p.rows = a->rows > 0 ? a->rows : INT_MAX;
    p.max_blocks = a->max_blocks; p.num_blocks = a->num_blocks; p.block_size = a->block_size; p.shift = shift;
    p.scale_log2 = a->scale * 1.4426950408889634f; p.causal = a->causal != 0;
    p.counters = static_cast<int*>(workspace);
    p.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + WS_COUNTERS);
    p.status = device_status_word();
    if (!p.status) return -1;
    // a tile of the cache as lines of 128 bytes: [blocks * heads][block_size * head_dim / 128][128]
    CUtensorMap tmK, tmV;
    const uint64_t tile = static_cast<uint64_t>(a->block_size) * a->head_dim;
    const uint64_t dims[3] = {128, tile / 128, static_cast<uint64_t>(a->num_blocks) * a->kv_heads}, strides[2] = {128, tile};
    const int halves = a->block_size < GROUP ? 2 : 1;
    const uint32_t box[3] = {128, static_cast<uint32_t>(GROUP / halves * a->head_dim / 128), 1};
    if (encode_tmap(&tmK, a->k_cache, 1, 3, dims, strides, box, true) != 0 || encode_tmap(&tmV, a->v_cache, 1, 3, dims, strides, box, true) != 0) return -1;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // Decided on the device, by two launches where max_query allows both: up to 8, 16 or 32 rows (the smallest that covers max_query,
    // or one token where max_query is beyond few_rows) the kernel for few rows, more than that the tcgen05 kernel.
    const long long most = static_cast<long long>(a->max_query) * p.group;
    const int limit = few_rows(a->head_dim);
    const int few = static_cast<int>(most <= limit ? most : p.group <= limit ? p.group : 0);
    p.cost = 2; p.unsplit = 8;               // an item's end takes about as long as two units' copies; a join takes 4 us, eight units 3
    const bool half = a->dtype == PYC_DTYPE_F16;
    const int upto = few <= 8 ? 8 : few <= 16 ? 16 : 32;
    if (few > 0) {
        p.rows_above = 0; p.rows_upto = upto;
        int rc;
#define B200_SHORT(D, NQ) (half ? launch_short<__half, D, NQ>(tmK, tmV, p, halves, s) : launch_short<__nv_bfloat16, D, NQ>(tmK, tmV, p, halves, s))
        if (a->head_dim == 128) rc = upto == 8 ? B200_SHORT(128, 1) : B200_SHORT(128, 2);
        else rc = upto == 8 ? B200_SHORT(64, 1) : upto == 16 ? B200_SHORT(64, 2) : B200_SHORT(64, 4);
#undef B200_SHORT
        if (rc != 0) return rc;
    }
    if (most <= limit) return 0;
    p.rows_above = few > 0 ? upto : 0; p.rows_upto = INT_MAX;
    return launch_paged_chunk(a->dtype, a->head_dim, p, a->k_cache, a->v_cache, s);
}

}  // extern "C"
