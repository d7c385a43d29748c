// Attention of a ragged batch of queries over the 8-bit paged key/value cache (layout and meaning: include/pyc_b200.h).
// PyC has no counterpart; the dense kernels are in attention.cu.
//
// This file: few query rows per key head (single new tokens, a few of them, grouped heads), which is bound by reading the
// cache.  A CTA walks the items of its stretch (paged_attention.cuh).  Each of its warps takes 32 keys of every unit
// and runs on its own: its own ring of TMA loads (keys and values, one copy each or two where a block is 16 tokens, into
// 128-byte swizzled shared memory), its own running maximum and sums in registers, no barrier with the other warps before
// the item's end.
//
// Products: mma m16n8k16, f16 x f16 -> f32, 16 rows of the tile at a time.  The codes become f16 exactly, one conversion per
// two codes, straight into operand registers:
//   * which head_dim value sits at which position of the contraction is free as long as queries and keys agree, so thread
//     (g = lane / 4, c = lane % 4) takes the D / 4 consecutive values from c * D / 4 of key g;
//   * for P V the same freedom holds for the columns: thread g takes the D / 8 consecutive values from g * D / 8 of the keys
//     2c, 2c + 1, 2c + 8, 2c + 9, which are the keys whose probabilities the score fragment leaves in this thread.
// So 16-byte shared-memory loads, conflict-free under the swizzle, feed the tensor cores without any exchange.
//
// Precision.  Queries are scaled per row by a power of two to [1, 2) before they become f16 (exact but for values below
// 2^-24 of the row's largest).  The value scale vs of a block joins the exponent, p' = 2^(score + log2 vs - m), with m the running
// maximum of score + log2 vs, so the f16 operand holds the weight with which the block's CODES enter the sum: its largest is
// near 1 whatever the scales, and f16's 11 bits hold (2^-12 relative error, 2^-25 absolute below 2^-14).  The softmax's
// weight is sum p' / vs in f32.  m only moves when it would grow by more than 2^8 (p' stays far below f16's 65504).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

#include "internal.h"
#include "paged_attention.cuh"
#include "ptx_sm100.cuh"

namespace b200 {
namespace {

constexpr int GROUP = 32;                    // keys that a warp takes at a time

// MT: 16-row tiles per item.
template <int D, int MT>
struct ShortCfg {
    static constexpr int NW = MT == 1 ? 4 : 8;                             // warps per CTA
    static constexpr int PER_SM = MT == 1 ? 3 : 1;                         // resident CTAs
    static constexpr int THREADS = NW * 32;
    static constexpr int UNIT = NW * GROUP;                                // keys per unit
    static constexpr int TILE = GROUP * D;                                 // bytes of a group's keys (or values)
    static constexpr int RING_BYTES = (MT == 1 ? 64 : 192) * 1024;
    static constexpr int STAGES = RING_BYTES / (NW * 2 * TILE);
    static constexpr int Q_OFF = RING_BYTES;
    static constexpr int Q_BYTES = MT * 16 * D * 2;
    static constexpr int ROW_OFF = Q_OFF + Q_BYTES;                        // float [MT * 16] row scales
    static constexpr int ML_OFF = ROW_OFF + MT * 16 * 4;                   // float [NW][MT * 16][2]
    static constexpr int INFO_OFF = ML_OFF + NW * MT * 16 * 8;             // float4 [NW][STAGES][2]
    static constexpr int BAR_OFF = INFO_OFF + NW * STAGES * 32;            // mbarriers [NW][STAGES]
    static constexpr int MISC_OFF = BAR_OFF + NW * STAGES * 8;             // long long [NW], int flag
    static constexpr int BYTES = MISC_OFF + NW * 8 + 16 + 1024;            // + alignment
    static_assert(NW * MT * 16 * D * 4 <= RING_BYTES, "the ring holds the warps' sums at an item's end");
    static_assert(STAGES >= 2 && STAGES <= 32 && (BYTES + 1024) * PER_SM <= 228 * 1024, "shared memory of an SM");
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

template <typename T, int D, int MT>
__global__ void __launch_bounds__(ShortCfg<D, MT>::THREADS, ShortCfg<D, MT>::PER_SM)
paged_short_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PagedParams p, int halves) {
    using SM = ShortCfg<D, MT>;
    constexpr int NW = SM::NW, THREADS = SM::THREADS, UNIT = SM::UNIT;
    constexpr int TILE = MT * 16, S = SM::STAGES, KC = D / 64, NT = D / 8;   // KC: 16-byte chunks of a key per thread; NT: column tiles
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c4 = lane & 3;
    float* row_scale = reinterpret_cast<float*>(smem + SM::ROW_OFF);
    float* warp_ml = reinterpret_cast<float*>(smem + SM::ML_OFF);
    float4* info = reinterpret_cast<float4*>(smem + SM::INFO_OFF) + w * S * 2;
    const uint32_t bars = smem_u32(smem + SM::BAR_OFF) + w * S * 8;
    const uint32_t ring = smem_u32(smem) + w * S * 2 * SM::TILE;
    const uint32_t q_frags = smem_u32(smem + SM::Q_OFF) + lane * 16;
    long long* scratch = reinterpret_cast<long long*>(smem + SM::MISC_OFF);
    int* flag = reinterpret_cast<int*>(scratch + NW);

    if (lane == 0) {
        for (int i = 0; i < S; ++i) mbar_init(bars + 8 * i, halves);
        fence_barrier_init();
        fence_proxy_async();
        if (w == 0) { prefetch_tmap(&tmK); prefetch_tmap(&tmV); }
    }
    PagedCursor c;
    const bool busy = paged_begin<THREADS, TILE, UNIT>(p, c, scratch, 1);
    __syncthreads();
    if (!busy) return;
    uint32_t phases = 0;                     // parity of each stage's next completion
    bool ok = true;
    // this thread's places in a stage: keys g (+ 8, 16, 24) and values 2c, 2c + 1 (+ 8, ...).  8 lines on the swizzle repeats: that
    // is 8 keys for D = 128 and 16 for D = 64, where 8 keys on the chunk's bit 2 (64 bytes) is the other one
    constexpr int ODD = D == 64 ? 64 : 0;
    uint32_t k_at[KC][2], v_at[2][2];
#pragma unroll
    for (int i = 0; i < KC; ++i) { k_at[i][0] = swizzled(g * D + c4 * (D / 4) + i * 16); k_at[i][1] = k_at[i][0] ^ ODD; }
#pragma unroll
    for (int i = 0; i < 2; ++i) { v_at[i][0] = swizzled((2 * c4 + i) * D + g * NT); v_at[i][1] = v_at[i][0] ^ ODD; }

    for (long long u = c.lo; u < c.hi;) {
        const int j0 = static_cast<int>(u - c.item), j1 = static_cast<int>(min(static_cast<long long>(c.units), c.hi - c.item));
        const int row0 = c.t * TILE, rows = min(TILE, c.q.rows - row0);
        const int kend = paged_tile_end<TILE>(p, c.q, c.t);
        const int* table = p.table + static_cast<size_t>(c.r) * p.max_blocks;

        // ---- the ring.  A group lies in one block (halves = 1, block sizes from 32) or in two of 16 tokens (halves = 2).  Lane
        // (j - base) * halves + i holds id and scales of half i of unit j's group, and issues its copies.
        int base = j0, id = -1;
        float4 about = make_float4(0.0f, 0.0f, 1.0f, 0.0f);                  // key scale (0: masked), log2 of the value scale, 1 / it
        auto fetch = [&](int j) {
            base = j;
            const int mine = j + (halves == 2 ? lane >> 1 : lane);
            const long long key = static_cast<long long>(mine) * UNIT + w * GROUP + (halves == 2 ? (lane & 1) * 16 : 0);
            id = -1;
            if (mine < j1 && key < kend) {
                id = __ldg(table + (key >> p.shift));
                if (static_cast<unsigned>(id) >= static_cast<unsigned>(p.num_blocks)) id = -1;
            }
            about.x = 0.0f;
            if (id >= 0) {
                const size_t at = static_cast<size_t>(id) * p.kv_heads + c.h;
                const float vs = paged_clamp_scale(__ldg(p.v_scale + at));
                about = make_float4(paged_clamp_scale(__ldg(p.k_scale + at)), log2f(vs), 1.0f / vs, 0.0f);
            }
        };
        auto issue = [&](int j, int st) {    // warp-uniform
            if (j >= j1 || !ok) return;
            if ((j - base) * halves >= 32) fetch(j);
            const int i = lane - (j - base) * halves;
            if (i >= 0 && i < halves) {
                info[st * 2 + i] = about;
                if (halves == 1) info[st * 2 + 1] = about;
                if (id >= 0) {
                    const uint32_t bytes = SM::TILE / halves, dst = ring + st * 2 * SM::TILE + i * (SM::TILE / 2);
                    const int y = ((j * UNIT + w * GROUP + i * 16) & (p.block_size - 1)) * D / 128, z = id * p.kv_heads + c.h;
                    mbar_arrive_expect_tx(bars + 8 * st, 2 * bytes);
                    tma_load_3d(dst, &tmK, bars + 8 * st, 0, y, z);
                    tma_load_3d(dst + SM::TILE, &tmV, bars + 8 * st, 0, y, z);
                } else mbar_arrive(bars + 8 * st);
            }
        };
        fetch(j0);
#pragma unroll 1
        for (int i = 0; i < S; ++i) issue(j0 + i, i);

        // ---- queries to f16 operand order: 16 threads per row, D / 16 values each
#pragma unroll
        for (int part = 0; part < TILE * 16 / THREADS; ++part) {
            const int row = part * (THREADS / 16) + (threadIdx.x >> 4), mt = row >> 4, x = threadIdx.x & 15;
            constexpr int NV = D / 16;
            float v[NV];
            float amax = 0.0f;
            bool finite = true;
            if (row < rows) {
                const int token = (row0 + row) / p.group, head = c.h * p.group + (row0 + row - token * p.group);
                const T* src = static_cast<const T*>(p.q) + (static_cast<size_t>(c.q.start) + token) * p.q_stride + static_cast<size_t>(head) * D + x * NV;
                uint32_t wd[NV / 2];
                if constexpr (NV == 8) *reinterpret_cast<uint4*>(wd) = __ldg(reinterpret_cast<const uint4*>(src));
                else *reinterpret_cast<uint2*>(wd) = __ldg(reinterpret_cast<const uint2*>(src));
#pragma unroll
                for (int i = 0; i < NV / 2; ++i) {
                    const float2 f = unpack2<T>(wd[i]);
                    v[2 * i] = f.x; v[2 * i + 1] = f.y;
                    amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
                    finite &= fabsf(f.x) < INFINITY && fabsf(f.y) < INFINITY;
                }
            } else {
#pragma unroll
                for (int i = 0; i < NV; ++i) v[i] = 0.0f;
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o, 16));
            const unsigned all = __ballot_sync(0xffffffffu, finite);
            const bool row_finite = ((all >> (lane & 16)) & 0xffffu) == 0xffffu;
            // 2^-e brings the largest to [1, 2) (at the ends of the range, where 2^e or 2^-e would be subnormal, within [0, 4))
            const int e = amax > 0.0f && row_finite ? min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, -126), 126) : 0;
            const float down = exp2_int(-e);
            if (x == 0) row_scale[row] = row_finite ? exp2_int(e) * p.scale_log2 : __int_as_float(0x7fffffff);
            const int r16 = row & 15;
#pragma unroll
            for (int i = 0; i < NV; i += 2) {
                const int d = x * NV + i;
                const int cc = d / (D / 4), j = (d % (D / 4)) / 4, pos = d & 3;
                const __half2 h = __floats2half2_rn(v[i] * down, v[i + 1] * down);
                const int reg = (r16 >= 8 ? 1 : 0) + (pos >= 2 ? 2 : 0);
                *reinterpret_cast<__half2*>(smem + SM::Q_OFF + ((((mt * (D / 16) + j) * 32) + (r16 & 7) * 4 + cc) * 4 + reg) * 4) = h;
            }
        }
        __syncthreads();

        int lim[MT][2];
        float qs[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = mt * 16 + i * 8 + g;
                lim[mt][i] = row < rows ? paged_limit(p, c.q, (row0 + row) / p.group) : kend;
                qs[mt][i] = row_scale[row];
            }
        const int all_see = paged_limit(p, c.q, row0 / p.group);             // keys that every row sees

        float o[MT][NT][4], m[MT][2], l[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int i = 0; i < 2; ++i) { m[mt][i] = -INFINITY; l[mt][i] = 0.0f; }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[mt][n][i] = 0.0f;
        }

        int st = 0;
#pragma unroll 1
        for (int j = j0; j < j1; ++j) {
            __syncwarp();
            const float4 in0 = info[st * 2], in1 = info[st * 2 + 1];
            if (ok) {
                ok = __all_sync(0xffffffffu, mbar_wait(bars + 8 * st, (phases >> st) & 1, p.status, 0x61));
                phases ^= 1u << st;
            }
            if (ok && (in0.x > 0.0f || in1.x > 0.0f)) {
                const uint32_t kt = ring + st * 2 * SM::TILE;
                const int key0 = j * UNIT + w * GROUP;
                float s[MT][4][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int t = 0; t < 4; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[mt][t][i] = 0.0f;
#pragma unroll
                for (int i = 0; i < KC; ++i) {
                    uint4 kk[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t) kk[t] = lds128(kt + k_at[i][t & 1] + t * 8 * D);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        uint32_t b[4][2];
#pragma unroll
                        for (int t = 0; t < 4; ++t) e4m3x4_to_f16x4(x == 0 ? kk[t].x : x == 1 ? kk[t].y : x == 2 ? kk[t].z : kk[t].w, b[t][0], b[t][1]);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            const uint4 qa = lds128(q_frags + (mt * (D / 16) + i * 4 + x) * 512);
                            const uint32_t a[4] = {qa.x, qa.y, qa.z, qa.w};
#pragma unroll
                            for (int t = 0; t < 4; ++t) mma_f16(s[mt][t], a, b[t][0], b[t][1]);
                        }
                    }
                }
                const bool cut = key0 + GROUP > all_see || in0.x == 0.0f || in1.x == 0.0f;      // some row does not see some key of the group
                uint32_t pa[MT][2][4];
                bool moved = false;
                float alpha[MT][2];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float f0 = qs[mt][i] * in0.x, f1 = qs[mt][i] * in1.x;
                        float x[8];
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            x[2 * t] = fmaf(s[mt][t][2 * i], t < 2 ? f0 : f1, t < 2 ? in0.y : in1.y);
                            x[2 * t + 1] = fmaf(s[mt][t][2 * i + 1], t < 2 ? f0 : f1, t < 2 ? in0.y : in1.y);
                        }
                        if (cut) {
                            const int left = lim[mt][i] - key0 - 2 * c4;
#pragma unroll
                            for (int t = 0; t < 4; ++t) {
                                const bool gone = (t < 2 ? in0.x : in1.x) == 0.0f;
                                if (gone || t * 8 >= left) x[2 * t] = -INFINITY;
                                if (gone || t * 8 + 1 >= left) x[2 * t + 1] = -INFINITY;
                            }
                        }
                        float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                        const bool move = mx > m[mt][i] + 8.0f;              // also from -inf
                        alpha[mt][i] = move ? ex2_approx(m[mt][i] - mx) : 1.0f;
                        if (move) m[mt][i] = mx;
                        moved |= move;
                        const float ref = m[mt][i] == -INFINITY ? 0.0f : m[mt][i];
#pragma unroll
                        for (int t = 0; t < 8; ++t) x[t] = ex2_approx(x[t] - ref);
                        l[mt][i] = fmaf((x[0] + x[1]) + (x[2] + x[3]), in0.z, fmaf((x[4] + x[5]) + (x[6] + x[7]), in1.z, l[mt][i] * alpha[mt][i]));
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            const __half2 h = __floats2half2_rn(x[2 * t], x[2 * t + 1]);
                            pa[mt][t >> 1][(t & 1) * 2 + i] = *reinterpret_cast<const uint32_t*>(&h);
                        }
                    }
                }
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[mt][n][i] *= alpha[mt][i >> 1];
                }
                // values, 16 keys at a time: rows 2c, 2c + 1, 2c + 8, 2c + 9, D / 8 codes each
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t v[4][NT / 4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t a = kt + SM::TILE + v_at[i & 1][i >> 1] + (half * 16 + (i >> 1) * 8) * D;
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
                        // bytes of two keys side by side: (key, key + 1) for columns 4x, 4x + 1 | 4x + 2, 4x + 3
                        uint32_t b0[4], b1[4];
                        e4m3x4_to_f16x4(prmt(v[0][x], v[1][x], 0x5140), b0[0], b0[1]);
                        e4m3x4_to_f16x4(prmt(v[0][x], v[1][x], 0x7362), b0[2], b0[3]);
                        e4m3x4_to_f16x4(prmt(v[2][x], v[3][x], 0x5140), b1[0], b1[1]);
                        e4m3x4_to_f16x4(prmt(v[2][x], v[3][x], 0x7362), b1[2], b1[3]);
#pragma unroll
                        for (int y = 0; y < 4; ++y)
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) mma_f16(o[mt][4 * x + y], pa[mt][half], b0[y], b1[y]);
                    }
                    if (own_nan) {                                           // NaN values in a group that not every row sees whole: only to the rows that see them
                        for (int k = 0; k < 16; ++k) {
                            const int key = key0 + half * 16 + k;
                            if (key >= kend) break;
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int y = 0; y < 2; ++y) {
                                    uint32_t byte;
                                    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(byte) : "r"(kt + SM::TILE + swizzled((half * 16 + k) * D + (2 * c4 + y) * NT + n)));
                                    if ((byte & 127u) == 127u) {
#pragma unroll
                                        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                                            for (int i = 0; i < 2; ++i)
                                                if (key < lim[mt][i]) o[mt][n][2 * i + y] = __int_as_float(0x7fffffff);
                                    }
                                }
                        }
                    }
                }
            }
            __syncwarp();
            issue(j + S, st);
            st = st + 1 == S ? 0 : st + 1;
        }

        // ---- the item's end: the warps' sums meet in the ring's memory (all copies have landed and been read)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                l[mt][i] += __shfl_xor_sync(0xffffffffu, l[mt][i], 1);
                l[mt][i] += __shfl_xor_sync(0xffffffffu, l[mt][i], 2);
            }
        __syncthreads();
        float* sums = reinterpret_cast<float*>(smem);                        // [NW][TILE][D]
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = mt * 16 + i * 8 + g;
                if (row < rows) {
                    float* dst = sums + (static_cast<size_t>(w) * TILE + row) * D + 2 * c4 * NT;
#pragma unroll
                    for (int y = 0; y < 2; ++y)
#pragma unroll
                        for (int n = 0; n < NT; n += 4)
                            *reinterpret_cast<float4*>(dst + y * NT + n) = make_float4(o[mt][n][2 * i + y], o[mt][n + 1][2 * i + y], o[mt][n + 2][2 * i + y], o[mt][n + 3][2 * i + y]);
                    if (c4 == 0) { warp_ml[(w * TILE + row) * 2] = m[mt][i]; warp_ml[(w * TILE + row) * 2 + 1] = l[mt][i]; }
                }
            }
        __syncthreads();
        const bool whole = j0 == 0 && j1 == c.units;
        float* part = p.partials + (static_cast<size_t>(blockIdx.x) * 2 + (j0 == 0 ? 1 : 0)) * (static_cast<size_t>(TILE) * (D + 2));
        for (int e = threadIdx.x; e < rows * (D / 2); e += THREADS) {
            const int row = e / (D / 2), d = (e % (D / 2)) * 2;
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < NW; ++i) mx = fmaxf(mx, warp_ml[(i * TILE + row) * 2]);
            const float ref = mx == -INFINITY ? 0.0f : mx;
            float sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                const float f = ex2_approx(warp_ml[(i * TILE + row) * 2] - ref);
                const float2 x = *reinterpret_cast<const float2*>(sums + (static_cast<size_t>(i) * TILE + row) * D + d);
                sum = fmaf(warp_ml[(i * TILE + row) * 2 + 1], f, sum);
                o0 = fmaf(x.x, f, o0); o1 = fmaf(x.y, f, o1);
            }
            if (whole) paged_finish2<T, D>(p, c, row0 + row, d, o0, o1, ref, sum);
            else {
                __stcg(reinterpret_cast<float2*>(part + row * D + d), make_float2(o0, o1));
                if (d == 0) { __stcg(part + TILE * D + row, mx); __stcg(part + TILE * (D + 1) + row, sum); }
            }
        }
        __syncthreads();
        if (!whole) paged_join<T, D, THREADS, TILE>(p, c, rows, row0, sums, flag);
        fence_proxy_async();                                                 // the ring's memory goes back to the copies
        __syncthreads();
        u = c.item + j1;
        if (u < c.hi) paged_next<TILE, UNIT>(p, c);
    }
    if (!ok) for (int i = 0; i < 2000; ++i) __nanosleep(1000);               // a wait has run out: let what is in flight land
}

template <typename T, int D, int MT>
int launch_short(const CUtensorMap& tmK, const CUtensorMap& tmV, const PagedParams& p, int halves, cudaStream_t s) {
    using SM = ShortCfg<D, MT>;
    auto kernel = paged_short_kernel<T, D, MT>;
    B200_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::BYTES));
    kernel<<<sm_count() * SM::PER_SM, SM::THREADS, SM::BYTES, s>>>(tmK, tmV, p, halves);
    B200_CUDA_OK(cudaGetLastError());
    count_launch();
    return 0;
}

constexpr size_t WS_COUNTERS = 4096;          // bytes: one int per CTA, at most 1024

// Two slots of [rows][D + 2] floats per CTA, for the larger of the two forms (one or two 16-row tiles).
size_t partial_bytes(int head_dim) {
    const int rows = std::max(ShortCfg<64, 1>::PER_SM * 16, ShortCfg<64, 2>::PER_SM * 32);
    return static_cast<size_t>(sm_count()) * rows * 2 * (head_dim + 2) * sizeof(float);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t pyc_b200_paged_attention_workspace_bytes(int requests, int max_query, int heads, int kv_heads, int head_dim) {
    if (requests < 1 || max_query < 1 || kv_heads < 1 || heads < kv_heads || heads % kv_heads || (head_dim != 64 && head_dim != 128)) return 0;
    return WS_COUNTERS + partial_bytes(head_dim);
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
    const long long most = static_cast<long long>(a->max_query) * p.group;
    p.rows_above = 0; p.rows_upto = INT_MAX;
    const bool wide = most > 16, half = a->dtype == PYC_DTYPE_F16;
#define B200_SHORT(D, MT) (half ? launch_short<__half, D, MT>(tmK, tmV, p, halves, s) : launch_short<__nv_bfloat16, D, MT>(tmK, tmV, p, halves, s))
    if (a->head_dim == 128) return wide ? B200_SHORT(128, 2) : B200_SHORT(128, 1);
    return wide ? B200_SHORT(64, 2) : B200_SHORT(64, 1);
#undef B200_SHORT
}

}  // extern "C"
