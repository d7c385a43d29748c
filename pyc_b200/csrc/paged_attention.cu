// Attention of a ragged batch of queries over the 8-bit paged key/value cache (layout and meaning: include/pyc_b200.h).
// PyC has no counterpart; the dense kernels are in attention.cu.
//
// One warp per (query, head): the lanes split the head dimension, keys one after the other with an online softmax.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"
#include "kv_cache.cuh"
#include "math.cuh"

namespace b200 {
namespace {

__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_float(__nv_bfloat16& o, float v) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_float(__half& o, float v) { o = __float2half_rn(v); }

__device__ __forceinline__ float clamp_scale(float s) { return fminf(fmaxf(s, 0x1p-40f), 0x1p72f); }

template <typename T, int D>
__global__ void __launch_bounds__(128)
paged_attention_kernel(pyc_b200_paged_attention_args p, int shift) {
    constexpr int VPL = D / 32;
    const int lane = threadIdx.x & 31;
    const int r = blockIdx.y;
    const long long w = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const int i = static_cast<int>(w / p.heads), h = static_cast<int>(w % p.heads);
    const int q0 = p.query_start[r], n = min(p.query_start[r + 1] - q0, p.max_query);
    if (i >= n) return;
    const int full = p.query_start[r + 1] - q0;
    const int len = static_cast<int>(min(static_cast<long long>(max(p.seq_lens[r], 0)), static_cast<long long>(p.max_blocks) * p.block_size));
    const int end = p.causal ? min(len, len - full + i + 1) : len;
    const int kh = h / (p.heads / p.kv_heads);
    const size_t row = static_cast<size_t>(q0) + i;
    float q[VPL], o[VPL];
    const T* qp = static_cast<const T*>(p.q) + row * p.q_stride + static_cast<size_t>(h) * D + lane * VPL;
    for (int d = 0; d < VPL; ++d) { q[d] = to_float(qp[d]); o[d] = 0.0f; }
    float m = -INFINITY, l = 0.0f;
    for (int j = 0; j < end; ++j) {
        const int id = p.block_table[static_cast<size_t>(r) * p.max_blocks + (j >> shift)];
        if (static_cast<unsigned>(id) >= static_cast<unsigned>(p.num_blocks)) continue;
        const size_t bh = static_cast<size_t>(id) * p.kv_heads + kh;
        const size_t at = (bh * p.block_size + (j & (p.block_size - 1))) * D + lane * VPL;
        float s = 0.0f;
        for (int d = 0; d < VPL; d += 2) {
            const float2 k = e4m3x2_to_float2(*reinterpret_cast<const uint16_t*>(static_cast<const uint8_t*>(p.k_cache) + at + d));
            s = fmaf(q[d], k.x, fmaf(q[d + 1], k.y, s));
        }
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= p.scale * clamp_scale(p.k_scale[bh]);
        const float mn = fmaxf(m, s);
        const float a = m == -INFINITY ? 0.0f : __expf(m - mn);
        const float e = __expf(s - mn), ev = e * clamp_scale(p.v_scale[bh]);
        l = l * a + e;
        for (int d = 0; d < VPL; d += 2) {
            const float2 v = e4m3x2_to_float2(*reinterpret_cast<const uint16_t*>(static_cast<const uint8_t*>(p.v_cache) + at + d));
            o[d] = o[d] * a + ev * v.x; o[d + 1] = o[d + 1] * a + ev * v.y;
        }
        m = mn;
    }
    T* op = static_cast<T*>(p.out) + row * p.out_stride + static_cast<size_t>(h) * D + lane * VPL;
    const bool none = l == 0.0f;
    for (int d = 0; d < VPL; ++d) from_float(op[d], none ? 0.0f : o[d] / l);
    if (p.lse && lane == 0) p.lse[row * p.heads + h] = none ? -INFINITY : m + logf(l);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t pyc_b200_paged_attention_workspace_bytes(int requests, int max_query, int heads, int kv_heads, int head_dim) {
    if (requests < 1 || max_query < 1 || kv_heads < 1 || heads < kv_heads || heads % kv_heads || (head_dim != 64 && head_dim != 128)) return 0;
    return 256;
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
    const size_t row = static_cast<size_t>(a->heads) * a->head_dim;
    pyc_b200_paged_attention_args p = *a;
    if (!p.q_stride) p.q_stride = row;
    if (!p.out_stride) p.out_stride = row;
    if (p.q_stride < row || p.out_stride < row || p.q_stride % 8 || p.out_stride % 8) { set_error("paged attention: row strides must be multiples of 8 and at least heads * head_dim"); return -1; }
    auto al = [](const void* x, size_t n) { return reinterpret_cast<uintptr_t>(x) % n == 0; };
    if (!al(p.q, 16) || !al(p.out, 16) || !al(p.k_cache, 16) || !al(p.v_cache, 16)) { set_error("paged attention: pointers must be 16-byte aligned"); return -1; }
    const size_t need = pyc_b200_paged_attention_workspace_bytes(a->requests, a->max_query, a->heads, a->kv_heads, a->head_dim);
    if (workspace_bytes < need) { set_error("paged attention: workspace of %zu bytes needed, %zu given", need, workspace_bytes); return -1; }
    if (!al(workspace, 256)) { set_error("paged attention: workspace must be 256-byte aligned"); return -1; }
    const dim3 grid(static_cast<unsigned>((static_cast<long long>(a->max_query) * a->heads + 3) / 4), a->requests);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->dtype == PYC_DTYPE_BF16) {
        if (a->head_dim == 128) paged_attention_kernel<__nv_bfloat16, 128><<<grid, 128, 0, s>>>(p, shift);
        else paged_attention_kernel<__nv_bfloat16, 64><<<grid, 128, 0, s>>>(p, shift);
    } else {
        if (a->head_dim == 128) paged_attention_kernel<__half, 128><<<grid, 128, 0, s>>>(p, shift);
        else paged_attention_kernel<__half, 64><<<grid, 128, 0, s>>>(p, shift);
    }
    B200_CUDA_OK(cudaGetLastError());
    count_launch();
    return 0;
}

}  // extern "C"
