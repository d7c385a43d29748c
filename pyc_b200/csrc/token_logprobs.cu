// Log probabilities of given tokens, entropy and the top alternatives from rows of logits, and the gradient
// (formulas and meaning: include/pyc_b200.h).  PyC has no counterpart; the row softmax is in elementwise.cu.
//
// One CTA per row.  The statistics take one pass with a running maximum m, s = sum e^(x - m) and t = sum (x - m) e^(x - m)
// (lse = m + ln s, entropy = ln s - t / s); each alternative takes another pass for the largest logit behind the previous one.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"
#include "math.cuh"

namespace b200 {
namespace {

constexpr int LT = 256;
constexpr int MAX_TOP = 32;

__device__ __forceinline__ float logit(const float* x, size_t i) { return x[i]; }
__device__ __forceinline__ float logit(const __nv_bfloat16* x, size_t i) { return __bfloat162float(x[i]); }
__device__ __forceinline__ float logit(const __half* x, size_t i) { return __half2float(x[i]); }
__device__ __forceinline__ void put(float* x, size_t i, float v) { x[i] = v; }
__device__ __forceinline__ void put(__nv_bfloat16* x, size_t i, float v) { x[i] = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half* x, size_t i, float v) { x[i] = __float2half_rn(v); }

struct Stats { float m, s, t; };
// Joins two running sums; a side that has seen nothing (m = -inf) contributes nothing.
__device__ __forceinline__ Stats join(const Stats& a, const Stats& b) {
    Stats c;
    c.m = fmaxf(a.m, b.m);
    const float da = a.m == c.m ? 0.0f : a.m - c.m, db = b.m == c.m ? 0.0f : b.m - c.m;
    const float ea = expf(da), eb = expf(db);
    c.s = a.s * ea + b.s * eb;
    // a side whose factor has vanished contributes nothing, however large its distance (0 * inf)
    c.t = (a.s * ea > 0.0f ? (a.t + a.s * da) * ea : 0.0f) + (b.s * eb > 0.0f ? (b.t + b.s * db) * eb : 0.0f);
    return c;
}

template <typename T>
__global__ void __launch_bounds__(LT)
token_logprobs_kernel(pyc_b200_token_logprobs_args p) {
    __shared__ Stats st[LT];
    __shared__ unsigned long long best[LT];
    __shared__ int broken;
    const size_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
    if (threadIdx.x == 0) broken = 0;
    __syncthreads();
    Stats a = {-INFINITY, 0.0f, 0.0f};
    bool bad = false;
    for (size_t i = threadIdx.x; i < p.vocab; i += LT) {
        const float v = logit(x, i);
        bad |= !(v < INFINITY);
        if (v == -INFINITY) continue;
        const Stats one = {v, 1.0f, 0.0f};
        a = join(a, one);
    }
    if (bad) broken = 1;
    st[threadIdx.x] = a;
    __syncthreads();
    for (int o = LT / 2; o > 0; o >>= 1) {
        if (threadIdx.x < o) st[threadIdx.x] = join(st[threadIdx.x], st[threadIdx.x + o]);
        __syncthreads();
    }
    const Stats all = st[0];
    const bool none = all.m == -INFINITY;
    const float nan = __int_as_float(0x7fffffff);
    // log probabilities are (x - m) - ln s: x - lse would lose ln s beside a large maximum
    const float ln_s = logf(all.s), lse = broken ? nan : none ? -INFINITY : all.m + ln_s;
    if (threadIdx.x == 0) {
        const int tok = p.tokens[row];
        const bool given = tok >= 0 && static_cast<size_t>(tok) < p.vocab;
        p.logprob[row] = broken ? nan : !given ? 0.0f : none ? -INFINITY : (logit(x, tok) - all.m) - ln_s;
        if (p.lse) p.lse[row] = lse;
        if (p.entropy) p.entropy[row] = broken ? nan : none ? 0.0f : ln_s - all.t / all.s;
    }
    // value, then lower index: one ordered 64-bit key; each round takes the largest key below the last one
    unsigned long long last = ~0ull;
    for (int k = 0; k < p.top_k; ++k) {
        unsigned long long mine = 0;
        for (size_t i = threadIdx.x; i < p.vocab; i += LT) {
            const unsigned u = __float_as_uint(logit(x, i) + 0.0f);
            const unsigned long long key = (static_cast<unsigned long long>(u & 0x80000000u ? ~u : u | 0x80000000u) << 32) | (0xffffffffu - static_cast<unsigned>(i));
            if (key < last && key > mine) mine = key;
        }
        best[threadIdx.x] = mine;
        __syncthreads();
        for (int o = LT / 2; o > 0; o >>= 1) {
            if (threadIdx.x < o && best[threadIdx.x + o] > best[threadIdx.x]) best[threadIdx.x] = best[threadIdx.x + o];
            __syncthreads();
        }
        last = best[0];
        if (threadIdx.x == 0) {
            const unsigned i = 0xffffffffu - static_cast<unsigned>(last);
            p.top_ids[row * p.top_k + k] = broken ? -1 : static_cast<int>(i);
            p.top_logprobs[row * p.top_k + k] = broken ? nan : none ? -INFINITY : (logit(x, i) - all.m) - ln_s;
        }
        __syncthreads();
    }
}

template <typename T>
__global__ void __launch_bounds__(LT)
token_logprobs_grad_kernel(pyc_b200_token_logprobs_grad_args p) {
    const size_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
    T* d = static_cast<T*>(p.grad_logits) + row * p.grad_stride;
    const float lse = p.lse[row];
    const float u = p.grad_logprob ? p.grad_logprob[row] : 0.0f, w = p.grad_entropy ? p.grad_entropy[row] : 0.0f;
    const float ent = w != 0.0f ? p.entropy[row] : 0.0f;
    const int tok = p.tokens[row];
    const bool given = tok >= 0 && static_cast<size_t>(tok) < p.vocab;
    const float c = (given ? u : 0.0f) + w * ent;
    for (size_t i = threadIdx.x; i < p.vocab; i += LT) {
        const float v = logit(x, i);
        const float lp = v - lse;
        float g = 0.0f;
        if (v != -INFINITY) g = -expf(lp) * (c + w * lp);
        if (given && i == static_cast<size_t>(tok) && lse != -INFINITY) g += u;
        put(d, i, g);
    }
}

bool logits_ok(pyc_dtype t, size_t rows, size_t vocab, size_t stride) {
    if (t != PYC_DTYPE_F32 && t != PYC_DTYPE_BF16 && t != PYC_DTYPE_F16) { set_error("token logprobs: unsupported dtype %d", static_cast<int>(t)); return false; }
    if (rows == 0 || vocab == 0 || rows > 0x7fffffffull || vocab > 0x7fffffffull) { set_error("token logprobs: rows and vocab must be 1 .. 2^31 - 1"); return false; }
    if (stride < vocab) { set_error("token logprobs: row stride %zu below vocab %zu", stride, vocab); return false; }
    return true;
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
    if (p.top_k < 0 || p.top_k > MAX_TOP || static_cast<size_t>(p.top_k) > p.vocab) { set_error("token logprobs: top_k %d is not in 0 .. min(%d, vocab)", p.top_k, MAX_TOP); return -1; }
    if (p.top_k && (!p.top_ids || !p.top_logprobs)) { set_error("token logprobs: top_k without top_ids and top_logprobs"); return -1; }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const unsigned grid = static_cast<unsigned>(p.rows);
    if (p.dtype == PYC_DTYPE_F32) token_logprobs_kernel<float><<<grid, LT, 0, s>>>(p);
    else if (p.dtype == PYC_DTYPE_BF16) token_logprobs_kernel<__nv_bfloat16><<<grid, LT, 0, s>>>(p);
    else token_logprobs_kernel<__half><<<grid, LT, 0, s>>>(p);
    B200_CUDA_OK(cudaGetLastError());
    count_launch();
    return 0;
}

int pyc_b200_token_logprobs_backward(const pyc_b200_token_logprobs_grad_args* a, void* stream) {
    if (!a || !a->logits || !a->tokens || !a->lse || !a->grad_logits) { set_error("token logprobs backward: NULL argument"); return -1; }
    if (a->grad_entropy && !a->entropy) { set_error("token logprobs backward: grad_entropy without entropy"); return -1; }
    pyc_b200_token_logprobs_grad_args p = *a;
    if (!p.row_stride) p.row_stride = p.vocab;
    if (!p.grad_stride) p.grad_stride = p.vocab;
    if (!logits_ok(p.dtype, p.rows, p.vocab, p.row_stride) || !logits_ok(p.dtype, p.rows, p.vocab, p.grad_stride)) return -1;
    if (p.grad_logits == p.logits && p.grad_stride != p.row_stride) { set_error("token logprobs backward: in place needs equal strides"); return -1; }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const unsigned grid = static_cast<unsigned>(p.rows);
    if (p.dtype == PYC_DTYPE_F32) token_logprobs_grad_kernel<float><<<grid, LT, 0, s>>>(p);
    else if (p.dtype == PYC_DTYPE_BF16) token_logprobs_grad_kernel<__nv_bfloat16><<<grid, LT, 0, s>>>(p);
    else token_logprobs_grad_kernel<__half><<<grid, LT, 0, s>>>(p);
    B200_CUDA_OK(cudaGetLastError());
    count_launch();
    return 0;
}

}  // extern "C"
