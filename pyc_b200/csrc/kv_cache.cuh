// What the cache's writer and readers share: e4m3 codes and the block scales.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {

// log2 of the block size (16, 32, 64 or 128), or -1.
int kv_block_shift(int block_size);

constexpr int KV_SCALE_EXP_MIN = -32, KV_SCALE_EXP_MAX = 64;

// 2^e for e in [-126, 127], exactly.
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }

// Two e4m3 codes (low byte first) as f16: exact, NaN stays NaN.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
    uint32_t h;
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(h) : "r"(two));
    return h;
}
// Four codes: the two low ones and the two high ones.
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t four, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(four));
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t two) {
    const uint32_t h = e4m3x2_to_f16x2(two);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Exponent of the smallest power of two s with amax / s <= 448 = 1.75 * 2^8, within the range that scales may take.
__device__ __forceinline__ int kv_scale_exponent(float amax) {
    if (!(amax > 0.0f)) return KV_SCALE_EXP_MIN;
    const uint32_t b = __float_as_uint(amax);
    // subnormal amax has exponent field 0 and lands below the range's lower end anyway
    const int e = static_cast<int>(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, KV_SCALE_EXP_MIN), KV_SCALE_EXP_MAX);
}
// Exponent of the smallest power of two not below a scale that is already there; nonsense (NaN, <= 0) gives the range's lower end.
__device__ __forceinline__ int kv_exponent_of_scale(float s) {
    if (!(s > 0.0f)) return KV_SCALE_EXP_MIN;
    const uint32_t b = __float_as_uint(s);
    const int e = static_cast<int>(b >> 23) - 127 + ((b & 0x7fffffu) ? 1 : 0);
    return min(max(e, KV_SCALE_EXP_MIN), KV_SCALE_EXP_MAX);
}

}  // namespace b200
