// Log probabilities of given tokens, entropy and the largest logits of rows of logits
// (include/dflash_batch.h).
#include "common.cuh"
#include "dflash_batch.h"

namespace dflash {
namespace lp {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxTop = 32;
constexpr int kUnroll = 4;        // 16-byte loads a thread has in flight
constexpr int kCandidates = 1024; // keys a CTA has room for ...
constexpr int kSettle = 128;      // ... and the number from which it raises its threshold to the best `top` of them
constexpr int kMaxSplit = 8;      // CTAs (one cluster) per row, at most
constexpr int kLanes = 4;         // lanes of a group of the first threshold: 64 groups, at least 2 kMaxTop
constexpr int kGroups = kThreads / kLanes;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Orders (value, id) by larger value, then lower id; -0 counts as 0.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long key_of(float x, int id) {
    return static_cast<unsigned long long>(order_of(x)) << 32 | static_cast<uint32_t>(~id);
}
__device__ __forceinline__ float value_of(unsigned long long key) {
    const uint32_t o = static_cast<uint32_t>(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

template <typename T>
struct Vec {  // a 16-byte load of logits
    static constexpr int N = 16 / sizeof(T);
    uint4 u;
    __device__ __forceinline__ float at(int i) const {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        if constexpr (N == 8) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        else return __uint_as_float(w[i]);
    }
    __device__ __forceinline__ float pick(int i) const {  // at() for an index that is not a constant
        const int k = N == 8 ? i >> 1 : i;
        const uint32_t w = k & 2 ? (k & 1 ? u.w : u.z) : (k & 1 ? u.y : u.x);
        if constexpr (N == 8) return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
        else return __uint_as_float(w);
    }
    __device__ __forceinline__ void hide() {  // -inf everywhere: counts as nothing
        const uint32_t v = N == 8 ? 0xff80ff80u : 0xff800000u;
        u = make_uint4(v, v, v, v);
    }
};
__device__ __forceinline__ float scalar(const uint16_t* p) { return bf16_bits_to_float(*p); }
__device__ __forceinline__ float scalar(const float* p) { return *p; }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Running maximum m (in logits), l = sum 2^((x - m) log2 e) and w = the same sum weighted by (x - m) log2 e.
struct Sums {
    float m, l, w;
    __device__ __forceinline__ void raise(float to) {  // m becomes the larger `to`
        const float d = (m - to) * kLog2e;             // may be -inf, as may l d: far below `to`, or nothing yet
        const float f = ex2(d);
        w = f == 0.f ? 0.f : f * fmaf(l, d, w);        // a weight of 0 takes no part (0 x inf would be NaN)
        l *= f;
        m = to;
    }
    __device__ __forceinline__ void add(float x) {     // x <= m or NaN
        const float d = (x - m) * kLog2e, e = ex2(d);
        l += e;
        w = fmaf(e, fmaxf(d, -1e30f), w);              // a weight of 0 takes no part, -inf logits included
    }
    __device__ __forceinline__ void join(const Sums& o) {
        Sums b = o;
        if (b.m > m) raise(b.m);
        else if (m > b.m) b.raise(m);
        l += b.l;
        w += b.w;
    }
};

struct Shared {
    unsigned long long keys[kCandidates];
    unsigned long long best[kMaxTop], picked[kMaxTop];  // the largest keys, in order
    unsigned long long joined[kMaxSplit * kMaxTop], parts[2 * kMaxSplit];  // in the first CTA, from all
    unsigned long long threshold;                       // keys above it are collected
    Sums sums[kWarps];
    uint32_t groups[kGroups];
    int count, found;
};

// The k-th largest of the first n keys in shared memory (n >= k >= 1): bisection on the key, a block
// vote per step.
__device__ unsigned long long kth_key(const unsigned long long* keys, int n, int k) {
    unsigned long long lo = 0;  // at least k keys are >= lo
    for (int bit = 63; bit >= 0; --bit) {
        const unsigned long long mid = lo | 1ull << bit;
        int c = 0;
        for (int i0 = 0; i0 < n; i0 += kThreads) {
            const int i = i0 + threadIdx.x;
            c += __syncthreads_count(i < n && keys[i] >= mid);
        }
        if (c >= k) lo = mid;
    }
    return lo;
}

// Writes the k largest of n distinct keys to out in order (fewer if n < k, then 0): each key's place is the
// number of keys above it.
__device__ void ranked(const unsigned long long* keys, int n, int k, unsigned long long* out) {
    for (int i = threadIdx.x; i < k; i += kThreads) out[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const unsigned long long mine = keys[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += keys[j] > mine;
        if (r < k) out[r] = mine;
    }
    __syncthreads();
}

// The k largest of the first n keys collected, in order, to s.best (n < k: then 0).
__device__ void largest(Shared& s, int n, int k) {
    __syncthreads();
    if (n <= kThreads) {
        ranked(s.keys, n, k, s.best);
        return;
    }
    const unsigned long long kth = kth_key(s.keys, n, k);
    if (threadIdx.x == 0) s.found = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads)
        if (s.keys[i] >= kth) s.picked[atomicAdd(&s.found, 1)] = s.keys[i];  // exactly k: keys are distinct
    __syncthreads();
    ranked(s.picked, k, k, s.best);
}

// Stores to the same place in the cluster's first CTA.
__device__ __forceinline__ void put(unsigned long long* at, unsigned long long v) {
    asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(map_to_rank(smem_u32(at), 0)), "l"(v) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// One pass over a row, split over the CTAs of a cluster in runs of 16-byte loads (the elements before the
// first 16-byte border go to the first CTA, those behind the last to the last).  Each thread keeps its own
// maximum and sums, raised once per kUnroll loads.  The alternatives are collected in the same pass: the
// first loads give a threshold (the top-th largest of the maxima of kGroups groups of threads, so at least
// `top` logits reach it), from then on only logits above it are looked at, a vector at a time.  Once more than
// kSettle have been found the threshold is the top-th of those; where even kCandidates had no room for a
// round's (a row that ascends), the round is looked at again under the new threshold.
// 509 bf16 rows of 248320 logits with eight alternatives take 91 us in a graph (2.8 TB/s; HBM alone would take 39): bound by
// issue (a conversion, a comparison, an exponential and two sums for each logit), by two block barriers a round with no load
// in flight, and by uneven SMs (509 rows are one wave of CTAs, three rows on some SMs and four on others).  Few rows are bound
// by latency: 8 of them 14.7 us.
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) logprobs_kernel(
    const T* __restrict__ logits, long long ld, int vocab, const int32_t* __restrict__ tokens, int n, int top,
    float* __restrict__ token_logprobs, float* __restrict__ entropy, int32_t* __restrict__ top_ids,
    float* __restrict__ top_logprobs) {
    __shared__ Shared s;
    constexpr int N = Vec<T>::N;
    pdl_wait();
    pdl_launch_dependents();
    const int split = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_rank());
    const int row = blockIdx.x / split, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const T* x = logits + (long long)row * ld;
    int token = -1;                    // the first tokens and their logits are asked for early
    float token_at = 0.f;
    if (rank == 0 && token_logprobs && tid < n) {
        token = tokens[(long long)row * n + tid];
        if (token >= 0 && token < vocab) token_at = scalar(x + token);
    }
    if (split > 1) cluster_arrive();
    const int lead = min(vocab, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(T)));
    const int vecs = (vocab - lead) / N;
    const int v0 = static_cast<int>((long long)vecs * rank / split), v1 = static_cast<int>((long long)vecs * (rank + 1) / split);
    const uint4* body = reinterpret_cast<const uint4*>(x + lead);
    const int tail = lead + vecs * N;  // first element behind the vectors
    Sums a{-3.402823466e38f, 0.f, 0.f};
    float edge = -INFINITY;            // a scalar element of the row's ends, for some threads of the end CTAs
    int edge_id = -1;
    if (rank == 0 && tid < lead) edge_id = tid;
    if (rank == split - 1 && tid >= kThreads - 32 && tail + tid - (kThreads - 32) < vocab) edge_id = tail + tid - (kThreads - 32);
    if (edge_id >= 0) edge = scalar(x + edge_id);
    if (tid == 0) {
        s.count = 0;
        s.threshold = 0;
    }
    __syncthreads();
    unsigned long long threshold = 0;
    float reach = -INFINITY;           // value of the threshold
    const auto collect = [&](float v, int id) {
        const unsigned long long key = key_of(v, id);
        if (v >= reach && key > threshold) {
            const int at = atomicAdd(&s.count, 1);
            if (at < kCandidates) s.keys[at] = key;
        }
    };
    const int per = kThreads * kUnroll;
    const int rounds = max(1, (v1 - v0 + per - 1) / per);
    for (int r = 0; r < rounds; ++r) {
        Vec<T> v[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int i = v0 + (r * kUnroll + u) * kThreads + tid;
            if (i < v1) v[u].u = __ldcs(body + i);
            else v[u].hide();
        }
        float peak[kUnroll], m = r == 0 ? edge : -INFINITY;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            peak[u] = v[u].at(0);
#pragma unroll
            for (int i = 1; i < N; ++i) peak[u] = fmaxf(peak[u], v[u].at(i));
            m = fmaxf(m, peak[u]);
        }
        if (m > a.m) a.raise(m);
        if (r == 0) a.add(edge);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int i = 0; i < N; ++i) a.add(v[u].at(i));
        if (top == 0) continue;
        if (r == 0) {  // the first threshold
            float g = m;
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
            if ((tid & (kLanes - 1)) == 0) s.groups[tid / kLanes] = order_of(g);
            __syncthreads();
            if (tid < kGroups) {
                const uint32_t mine = s.groups[tid];
                int above = 0;
                for (int j = 0; j < kGroups; ++j) above += s.groups[j] > mine || (s.groups[j] == mine && j < tid);
                if (above == top - 1) s.threshold = static_cast<unsigned long long>(mine) << 32;  // below every key of the value
            }
            __syncthreads();
            threshold = s.threshold;
            reach = value_of(threshold);
        }
        // collect, until everything above the threshold fits
        int base = s.count;  // keys of earlier rounds
        while (true) {
            __syncthreads();  // base is read
            if (r == 0 && edge_id >= 0) collect(edge, edge_id);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int i = v0 + (r * kUnroll + u) * kThreads + tid;
                if (peak[u] >= reach && i < v1) {  // seldom
                    uint32_t found = 0;
#pragma unroll
                    for (int e = 0; e < N; ++e) found |= (v[u].at(e) >= reach ? 1u : 0u) << e;
                    while (found) {
                        const int e = __ffs(found) - 1;
                        found &= found - 1;
                        collect(v[u].pick(e), lead + i * N + e);
                    }
                }
            }
            __syncthreads();
            const int found = s.count;
            if (found <= kSettle) break;
            const bool all = found <= kCandidates;
            largest(s, all ? found : kCandidates, top);
            threshold = s.best[top - 1];
            reach = value_of(threshold);
            if (all) {  // the best so far are all that is kept
                __syncthreads();
                if (tid < top) s.keys[tid] = s.best[tid];
                if (tid == 0) s.count = top;
                break;
            }
            // some keys found no room: those of earlier rounds that reach the new threshold stay, this round's
            // are collected again
            if (tid == 0) {
                int kept = 0;
                for (int e = 0; e < top; ++e)
                    for (int o = 0; o < base; ++o)
                        if (s.keys[o] == s.best[e]) s.picked[kept++] = s.best[e];
                for (int e = 0; e < kept; ++e) s.keys[e] = s.picked[e];
                s.count = kept;
                --threshold;
                s.threshold = threshold;
            }
            __syncthreads();
            threshold = s.threshold;
            base = s.count;
        }
    }
    // the warps' and the CTAs' sums and alternatives
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Sums b;
        b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
        b.l = __shfl_xor_sync(0xffffffffu, a.l, o);
        b.w = __shfl_xor_sync(0xffffffffu, a.w, o);
        a.join(b);
    }
    if (lane == 0) s.sums[warp] = a;
    __syncthreads();
    if (top > 0) largest(s, s.count, top);
    if (split > 1) {
        cluster_wait();  // every CTA of the cluster has started
        if (tid < top) put(&s.joined[rank * top + tid], s.best[tid]);
        if (tid == 0) {
            Sums t = s.sums[0];
            for (int i = 1; i < kWarps; ++i) t.join(s.sums[i]);
            put(&s.parts[2 * rank], static_cast<unsigned long long>(__float_as_uint(t.m)) << 32 | __float_as_uint(t.l));
            put(&s.parts[2 * rank + 1], __float_as_uint(t.w));
        }
        cluster_sync_all();
        if (rank != 0) return;
        if (top > 0) ranked(s.joined, split * top, top, s.best);
    }
    Sums t{-3.402823466e38f, 0.f, 0.f};
    if (split > 1) {
        for (int i = 0; i < split; ++i)
            t.join(Sums{__uint_as_float(static_cast<uint32_t>(s.parts[2 * i] >> 32)),
                        __uint_as_float(static_cast<uint32_t>(s.parts[2 * i])),
                        __uint_as_float(static_cast<uint32_t>(s.parts[2 * i + 1]))});
    } else {
        for (int i = 0; i < kWarps; ++i) t.join(s.sums[i]);
    }
    const bool none = !(t.l >= 0.5f && t.l < INFINITY);  // a NaN, a +inf, or nothing above -inf
    const float nan = __int_as_float(0x7fc00000), log_l = logf(t.l);
    if (tid == 0 && entropy) entropy[row] = none ? nan : log_l - t.w * kLn2 / t.l;
    if (token_logprobs)
        for (int j = tid; j < n; j += kThreads) {
            const int id = j == tid ? token : tokens[(long long)row * n + j];
            const float at = j == tid ? token_at : id >= 0 && id < vocab ? scalar(x + id) : 0.f;
            token_logprobs[(long long)row * n + j] = id < 0 ? 0.f : id >= vocab || none ? nan : at - t.m - log_l;
        }
    if (tid < top) {
        const unsigned long long key = s.best[tid];
        if (top_ids) top_ids[(long long)row * top + tid] = none ? -1 : static_cast<int>(~static_cast<uint32_t>(key));
        if (top_logprobs) top_logprobs[(long long)row * top + tid] = none ? nan : value_of(key) - t.m - log_l;
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
    if (vocab > 0x7fffffff - lp::kThreads)
        return fail(DFLASH_ERR_UNSUPPORTED, "dflash_logprobs: a vocabulary of %d", vocab);
    if (top > lp::kMaxTop || top > vocab)
        return fail(DFLASH_ERR_UNSUPPORTED, "dflash_logprobs: %d alternatives; at most %d and the vocabulary's %d", top,
                    lp::kMaxTop, vocab);
    if (reinterpret_cast<uintptr_t>(logits) % (type == DFLASH_LOGITS_BF16 ? 2 : 4))
        return fail(DFLASH_ERR_MISALIGNED, "dflash_logprobs: logits not aligned to their type");
    if (rows == 0) return DFLASH_OK;
    if (!top_ids && !top_logprobs) top = 0;
    if (n == 0) token_logprobs = nullptr;
    int dev = 0;
    DFLASH_CUDA_TRY(cudaGetDevice(&dev));
    // a cluster per row while all CTAs fit on the SMs at once (four each) and have a few loads per thread left: 8 rows of
    // 248320 take 49 us with one CTA, 30 with two, 14.7 with eight; 61 of 50021 19.8, 12.6 and (eight) 9.5; 509 of
    // 248320 91 with one and 97 with two
    int split = 1;
    while (split < lp::kMaxSplit && 2ll * split * rows <= 4ll * sm_count(dev) && vocab / (2 * split) >= 4096) split *= 2;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid(static_cast<unsigned>(rows) * split), block(lp::kThreads);
    cudaError_t e;
    if (type == DFLASH_LOGITS_BF16)
        e = launch_chained(lp::logprobs_kernel<uint16_t>, grid, block, 0, s, split, static_cast<const uint16_t*>(logits), ld,
                           vocab, tokens, n, top, token_logprobs, entropy, top_ids, top_logprobs);
    else
        e = launch_chained(lp::logprobs_kernel<float>, grid, block, 0, s, split, static_cast<const float*>(logits), ld,
                           vocab, tokens, n, top, token_logprobs, entropy, top_ids, top_logprobs);
    DFLASH_CUDA_TRY(e);
    return DFLASH_OK;
}
