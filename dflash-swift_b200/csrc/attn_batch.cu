// Decode attention of a batch of sequences over caches of 16, 8 or 4 bits, with an optional
// prefix that all of them share (include/dflash_batch.h).
#include "common.cuh"
#include "dflash_batch.h"

namespace dflash {
namespace attn {

constexpr int kThreads = 256;
constexpr int kHeads = 8;  // q heads of one kv head that a CTA serves

struct Args {
    const uint16_t* q;
    const uint16_t* gate;
    uint16_t* out;
    long long ld_q, ld_gate;
    kv::View cache, prefix;
    const int32_t* lengths;
    const int32_t* parents;
    int prefix_len, tokens, hq;
    float scale;
};

__device__ __forceinline__ float element(const uint8_t* codes, const uint16_t* scales, const uint16_t* biases, int64_t row,
                                         int d, int bits, int group, int e) {
    if (bits == 16) return bf16_bits_to_float(reinterpret_cast<const uint16_t*>(codes)[row * d + e]);
    const int64_t g = row * (d / group) + e / group;
    const int c = bits == 8 ? codes[row * d + e] : (codes[(row * d + e) / 2] >> (4 * (e & 1))) & 15;
    return fmaf(bf16_bits_to_float(scales[g]), static_cast<float>(c), bf16_bits_to_float(biases[g]));
}

// One CTA per (row, kv head, group of kHeads q heads): an online softmax over chunks of kThreads
// keys, a thread scoring one key, then a thread summing one element of p V.
__global__ void __launch_bounds__(kThreads) attn_batch_kernel(Args a) {
    extern __shared__ float smem[];
    const int d = a.cache.d, G = a.hq / a.cache.hkv;
    float* s_q = smem;                    // [kHeads][d]
    float* s_p = s_q + kHeads * d;        // [kHeads][kThreads]
    float* s_acc = s_p + kHeads * kThreads;  // [kHeads][d]
    __shared__ float s_m[kHeads], s_l[kHeads], s_corr[kHeads];
    pdl_wait();
    pdl_launch_dependents();
    const int r = blockIdx.x, seq = r / a.tokens, t = r - seq * a.tokens, head = blockIdx.y, g0 = blockIdx.z * kHeads;
    const int heads = min(kHeads, G - g0), tid = threadIdx.x;
    const int n = kv::block_start(a.lengths, seq, a.tokens, a.cache.max_len);
    if (n < 0) return;
    const uint32_t path = a.parents ? tree_walk(a.parents + (size_t)seq * a.tokens, t).path : 0u;
    const size_t h0 = (size_t)head * G + g0;
    for (int i = tid; i < heads * d; i += kThreads) {
        s_q[i] = bf16_bits_to_float(a.q[(size_t)r * a.ld_q + h0 * d + i]) * a.scale;
        s_acc[i] = 0.f;
    }
    if (tid < kHeads) {
        s_m[tid] = -INFINITY;
        s_l[tid] = 0.f;
    }
    const int total = a.prefix_len + n + t + 1;
    for (int c0 = 0; c0 < total; c0 += kThreads) {
        const int key = c0 + tid, own = key - a.prefix_len;
        const bool in_prefix = key < a.prefix_len;
        const bool seen = key < total && (in_prefix || !a.parents || own < n || ((path >> (own - n)) & 1u));
        const kv::View& c = in_prefix ? a.prefix : a.cache;
        const int64_t row = in_prefix ? kv::row_index(c, 0, head, key) : kv::row_index(c, seq, head, own);
        __syncthreads();
        float dot[kHeads];
        for (int g = 0; g < kHeads; ++g) dot[g] = 0.f;
        if (seen)
            for (int e = 0; e < d; ++e) {
                const float k = element(c.k, c.ks, c.kb, row, d, c.bits, c.group, e);
#pragma unroll
                for (int g = 0; g < kHeads; ++g) dot[g] = fmaf(g < heads ? s_q[g * d + e] : 0.f, k, dot[g]);
            }
        for (int g = 0; g < heads; ++g) s_p[g * kThreads + tid] = seen ? dot[g] : -INFINITY;
        __syncthreads();
        if (tid < heads) {
            float m = s_m[tid], l = 0.f;
            for (int j = 0; j < kThreads; ++j) m = fmaxf(m, s_p[tid * kThreads + j]);
            const float base = m == -INFINITY ? 0.f : m;
            for (int j = 0; j < kThreads; ++j) {
                const float p = __expf(s_p[tid * kThreads + j] - base);
                s_p[tid * kThreads + j] = p;
                l += p;
            }
            s_corr[tid] = __expf(s_m[tid] - base);
            s_l[tid] = s_l[tid] * s_corr[tid] + l;
            s_m[tid] = m;
        }
        __syncthreads();
        for (int i = tid; i < heads * d; i += kThreads) {
            const int g = i / d, e = i - g * d;
            float acc = s_acc[i] * s_corr[g];
            for (int j = 0; j < kThreads && c0 + j < total; ++j) {
                const int kj = c0 + j, oj = kj - a.prefix_len;
                if (kj >= a.prefix_len && a.parents && oj >= n && !((path >> (oj - n)) & 1u)) continue;
                const kv::View& cj = kj < a.prefix_len ? a.prefix : a.cache;
                const int64_t rj = kj < a.prefix_len ? kv::row_index(cj, 0, head, kj) : kv::row_index(cj, seq, head, oj);
                acc = fmaf(s_p[g * kThreads + j], element(cj.v, cj.vs, cj.vb, rj, d, cj.bits, cj.group, e), acc);
            }
            s_acc[i] = acc;
        }
    }
    __syncthreads();
    for (int i = tid; i < heads * d; i += kThreads) {
        float o = s_acc[i] / s_l[i / d];
        if (a.gate) o /= 1.f + __expf(-bf16_bits_to_float(a.gate[(size_t)r * a.ld_gate + h0 * d + i]));
        a.out[((size_t)r * a.hq + h0) * d + i] = kv::bf_bits(o);
    }
}

static int check(const dflash_kv_cache* cache, const dflash_kv_cache* prefix, int prefix_len, int tokens, int hq,
                 const char* who) {
    const int st = kv::check_cache(cache, who);
    if (st != DFLASH_OK) return st;
    if (tokens < 1 || tokens > cache->max_len || hq < 1 || hq % cache->kv_heads || prefix_len < 0)
        return fail(DFLASH_ERR_INVALID_ARGUMENT, "%s: bad arguments", who);
    if (hq / cache->kv_heads > 64 || (long long)cache->sequences * tokens > 0x7fffffffll / hq ||
        (long long)prefix_len + cache->max_len > 0x7fffffffll - 128)
        return fail(DFLASH_ERR_UNSUPPORTED, "%s: too many rows or keys, or more than 64 q heads per kv head", who);
    if (prefix_len > 0 && prefix) {
        const int sp = kv::check_cache(prefix, who);
        if (sp != DFLASH_OK) return sp;
        if (prefix->sequences != 1 || prefix->kv_heads != cache->kv_heads || prefix->head_dim != cache->head_dim ||
            prefix->bits != cache->bits || (cache->bits != 16 && prefix->group != cache->group) ||
            prefix_len > prefix->max_len)
            return fail(DFLASH_ERR_INVALID_ARGUMENT, "%s: the prefix must be one sequence in the cache's format, at least "
                        "prefix_len rows long", who);
    }
    return DFLASH_OK;
}

}  // namespace attn
}  // namespace dflash

extern "C" size_t dflash_stack_attn_decode_batch_workspace_bytes(const dflash_kv_cache* cache, int prefix_len, int tokens,
                                                                 int hq) {
    using namespace dflash;
    if (attn::check(cache, nullptr, prefix_len, tokens, hq, "dflash_stack_attn_decode_batch_workspace_bytes") != DFLASH_OK)
        return 0;
    return 16;
}

extern "C" int dflash_stack_attn_decode_batch(const dflash_bf16* q, long long ld_q, const dflash_bf16* gate,
                                              long long ld_gate, const dflash_kv_cache* cache, const int32_t* lengths,
                                              const dflash_kv_cache* prefix, int prefix_len, dflash_bf16* out, int tokens,
                                              int hq, float scale, const int32_t* parents, void* workspace,
                                              size_t workspace_bytes, dflash_stream_t stream) {
    using namespace dflash;
    const char* who = "dflash_stack_attn_decode_batch";
    const int st = attn::check(cache, prefix, prefix_len, tokens, hq, who);
    if (st != DFLASH_OK) return st;
    const int d = cache->head_dim, G = hq / cache->kv_heads;
    if (!q || !lengths || !out || (parents && tokens > kMaxTreeRows) || (prefix_len > 0 && !prefix) ||
        ld_q < (long long)hq * d || (gate && ld_gate < (long long)hq * d))
        return fail(DFLASH_ERR_INVALID_ARGUMENT, "%s: bad arguments", who);
    if (!kv::stride_ok(q, ld_q, 1) || (gate && !kv::stride_ok(gate, ld_gate, 1)) || !aligned16(out))
        return fail(DFLASH_ERR_MISALIGNED, "%s: q, gate, out and their row strides must be 16-byte aligned", who);
    const size_t need = dflash_stack_attn_decode_batch_workspace_bytes(cache, prefix_len, tokens, hq);
    if (!workspace || workspace_bytes < need || !aligned16(workspace))
        return fail(DFLASH_ERR_WORKSPACE, "%s: needs %zu bytes of 16-byte aligned workspace", who, need);
    attn::Args a{q, gate, out, ld_q, ld_gate, kv::view_of(*cache), prefix_len > 0 ? kv::view_of(*prefix) : kv::view_of(*cache),
                 lengths, parents, prefix_len, tokens, hq, scale};
    const size_t smem = sizeof(float) * (2 * attn::kHeads * d + attn::kHeads * attn::kThreads);
    const dim3 grid(cache->sequences * tokens, cache->kv_heads, (G + attn::kHeads - 1) / attn::kHeads);
    DFLASH_CUDA_TRY(launch_chained(attn::attn_batch_kernel, grid, dim3(attn::kThreads), smem,
                                   reinterpret_cast<cudaStream_t>(stream), 1, a));
    return DFLASH_OK;
}
