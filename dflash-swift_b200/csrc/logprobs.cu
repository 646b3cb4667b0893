// Log probabilities of given tokens, entropy and the largest logits of rows of logits
// (include/dflash_batch.h).
#include "common.cuh"
#include "dflash_batch.h"

namespace dflash {
namespace lp {

constexpr int kThreads = 512;
constexpr int kMaxTop = 32;

__device__ __forceinline__ float value(const uint16_t* p, long long i) { return bf16_bits_to_float(p[i]); }
__device__ __forceinline__ float value(const float* p, long long i) { return p[i]; }

// Orders (value, id) by larger value, then lower id; -0 counts as 0.
__device__ __forceinline__ unsigned long long key_of(float x, int id) {
    const uint32_t u = __float_as_uint(x + 0.f);
    const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
    return static_cast<unsigned long long>(o) << 32 | static_cast<uint32_t>(~id);
}
__device__ __forceinline__ float value_of(unsigned long long key) {
    const uint32_t o = static_cast<uint32_t>(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// One CTA per row: the maximum, then the sums, then `top` passes that each find the largest key
// below the last one.
template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const T* __restrict__ logits, long long ld, int vocab,
                                                            const int32_t* __restrict__ tokens, int n, int top,
                                                            float* __restrict__ token_logprobs, float* __restrict__ entropy,
                                                            int32_t* __restrict__ top_ids, float* __restrict__ top_logprobs) {
    __shared__ unsigned long long s_key[kThreads];
    __shared__ float s_a[kThreads], s_b[kThreads];
    pdl_wait();
    pdl_launch_dependents();
    const int row = blockIdx.x, tid = threadIdx.x;
    const T* x = logits + (long long)row * ld;
    float m = -INFINITY;
    for (int i = tid; i < vocab; i += kThreads) m = fmaxf(m, value(x, i));
    s_a[tid] = m;
    __syncthreads();
    for (int o = kThreads / 2; o > 0; o >>= 1) {
        if (tid < o) s_a[tid] = fmaxf(s_a[tid], s_a[tid + o]);
        __syncthreads();
    }
    m = s_a[0];
    __syncthreads();
    float l = 0.f, w = 0.f;  // sum e, sum e (x - m)
    for (int i = tid; i < vocab; i += kThreads) {
        const float y = value(x, i) - m, e = expf(y);
        l += e;
        w += e == 0.f ? 0.f : e * y;
    }
    s_a[tid] = l;
    s_b[tid] = w;
    __syncthreads();
    for (int o = kThreads / 2; o > 0; o >>= 1) {
        if (tid < o) {
            s_a[tid] += s_a[tid + o];
            s_b[tid] += s_b[tid + o];
        }
        __syncthreads();
    }
    l = s_a[0];
    w = s_b[0];
    const bool none = !(l >= 1.f && l < INFINITY);  // a NaN, a +inf, or nothing above -inf
    const float nan = __int_as_float(0x7fc00000), log_l = logf(l);
    if (tid == 0 && entropy) entropy[row] = none ? nan : log_l - w / l;
    if (token_logprobs)
        for (int j = tid; j < n; j += kThreads) {
            const int t = tokens[(long long)row * n + j];
            token_logprobs[(long long)row * n + j] = t < 0 ? 0.f : t >= vocab || none ? nan : value(x, t) - m - log_l;
        }
    unsigned long long last = ~0ull;
    for (int k = 0; k < top; ++k) {
        unsigned long long best = 0;
        if (!none)
            for (int i = tid; i < vocab; i += kThreads) {
                const unsigned long long key = key_of(value(x, i), i);
                if (key < last && key > best) best = key;
            }
        s_key[tid] = best;
        __syncthreads();
        for (int o = kThreads / 2; o > 0; o >>= 1) {
            if (tid < o && s_key[tid + o] > s_key[tid]) s_key[tid] = s_key[tid + o];
            __syncthreads();
        }
        last = s_key[0];
        __syncthreads();
        if (tid == 0) {
            if (top_ids) top_ids[(long long)row * top + k] = none ? -1 : static_cast<int>(~static_cast<uint32_t>(last));
            if (top_logprobs) top_logprobs[(long long)row * top + k] = none ? nan : value_of(last) - m - log_l;
        }
    }
}

}  // namespace lp
}  // namespace dflash

extern "C" int dflash_logprobs(const void* logits, int type, long long ld, int rows, int vocab, const int32_t* tokens, int n,
                               int top, float* token_logprobs, float* entropy, int32_t* top_ids, float* top_logprobs,
                               dflash_stream_t stream) {
    using namespace dflash;
    if ((!logits && rows > 0) || rows < 0 || vocab < 1 || ld < vocab || n < 0 || top < 0 || (token_logprobs && n > 0 && rows > 0 && !tokens))
        return fail(DFLASH_ERR_INVALID_ARGUMENT, "dflash_logprobs: bad arguments");
    if (type != DFLASH_LOGITS_BF16 && type != DFLASH_LOGITS_FP32)
        return fail(DFLASH_ERR_UNSUPPORTED, "dflash_logprobs: logits type %d; bf16 (0) or fp32 (1)", type);
    if (top > lp::kMaxTop || top > vocab)
        return fail(DFLASH_ERR_UNSUPPORTED, "dflash_logprobs: %d alternatives; at most %d and the vocabulary's %d", top,
                    lp::kMaxTop, vocab);
    if (reinterpret_cast<uintptr_t>(logits) % (type == DFLASH_LOGITS_BF16 ? 2 : 4))
        return fail(DFLASH_ERR_MISALIGNED, "dflash_logprobs: logits not aligned to their type");
    if (rows == 0) return DFLASH_OK;
    if (!top_ids && !top_logprobs) top = 0;
    if (n == 0) token_logprobs = nullptr;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid(rows), block(lp::kThreads);
    cudaError_t e;
    if (type == DFLASH_LOGITS_BF16)
        e = launch_chained(lp::logprobs_kernel<uint16_t>, grid, block, 0, s, 1, static_cast<const uint16_t*>(logits), ld,
                           vocab, tokens, n, top, token_logprobs, entropy, top_ids, top_logprobs);
    else
        e = launch_chained(lp::logprobs_kernel<float>, grid, block, 0, s, 1, static_cast<const float*>(logits), ld, vocab,
                           tokens, n, top, token_logprobs, entropy, top_ids, top_logprobs);
    DFLASH_CUDA_TRY(e);
    return DFLASH_OK;
}
