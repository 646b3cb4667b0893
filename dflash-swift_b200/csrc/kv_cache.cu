// Attention caches of a batch of sequences in 16, 8 or 4 bits (include/dflash_batch.h): the
// attention prep that writes them, the read-back and the move of accepted tree rows.  The
// attention over them is attn_batch.cu.
#include "common.cuh"
#include "dflash_batch.h"

namespace dflash {
namespace kv {

// dflash_kv_cache as the kernels take it.
struct View {
    uint8_t* k;
    uint8_t* v;
    uint16_t *ks, *kb, *vs, *vb;
    int sequences, hkv, max_len, d, bits, group;
};

inline View view_of(const dflash_kv_cache& c) {
    return View{static_cast<uint8_t*>(c.k), static_cast<uint8_t*>(c.v), c.k_scales, c.k_biases, c.v_scales, c.v_biases,
                c.sequences, c.kv_heads, c.max_len, c.head_dim, c.bits, c.group};
}

// Host check of a cache descriptor; DFLASH_OK or the status with its message set.
inline int check_cache(const dflash_kv_cache* c, const char* who) {
    if (!c || !c->k || !c->v || c->sequences < 1 || c->kv_heads < 1 || c->max_len < 1)
        return fail(DFLASH_ERR_INVALID_ARGUMENT, "%s: bad cache (null k or v, or an empty shape)", who);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(DFLASH_ERR_UNSUPPORTED, "%s: head dim %d not in {64,128,256}", who, c->head_dim);
    if (c->bits != 16 && c->bits != 8 && c->bits != 4)
        return fail(DFLASH_ERR_UNSUPPORTED, "%s: %d-bit cache; 16, 8 or 4", who, c->bits);
    if (c->bits != 16) {
        if ((c->group != 32 && c->group != 64 && c->group != 128) || c->group > c->head_dim)
            return fail(DFLASH_ERR_UNSUPPORTED, "%s: group %d not in {32,64,128} or above head dim %d", who, c->group,
                        c->head_dim);
        if (!c->k_scales || !c->k_biases || !c->v_scales || !c->v_biases)
            return fail(DFLASH_ERR_INVALID_ARGUMENT, "%s: a quantised cache needs scales and biases", who);
        if (((reinterpret_cast<uintptr_t>(c->k_scales) | reinterpret_cast<uintptr_t>(c->k_biases) |
              reinterpret_cast<uintptr_t>(c->v_scales) | reinterpret_cast<uintptr_t>(c->v_biases)) & 15u) != 0)
            return fail(DFLASH_ERR_MISALIGNED, "%s: scales and biases must be 16-byte aligned", who);
    }
    if (!aligned16(c->k) || !aligned16(c->v))
        return fail(DFLASH_ERR_MISALIGNED, "%s: k and v must be 16-byte aligned", who);
    if (c->sequences > 65535 || c->kv_heads > 65535)
        return fail(DFLASH_ERR_UNSUPPORTED, "%s: more than 65535 sequences or kv heads", who);
    return DFLASH_OK;
}

__device__ __forceinline__ uint16_t bf_bits(float v) {
    const __nv_bfloat16 h = __float2bfloat16_rn(v);
    return *reinterpret_cast<const uint16_t*>(&h);
}

__device__ __forceinline__ int64_t row_index(const View& c, int seq, int head, int row) {
    return ((int64_t)seq * c.hkv + head) * c.max_len + row;
}

// The block's first cache row, or -1 when the sequence takes no part (raising the device
// error when its block would not fit).
__device__ __forceinline__ int block_start(const int32_t* __restrict__ lengths, int seq, int tokens, int max_len) {
    const int n = lengths[seq];
    if (n < 0) return -1;
    if (n > max_len - tokens) {
        atomicOr(&g_device_error, DFLASH_DEVERR_POSITION);
        return -1;
    }
    return n;
}

// CH consecutive bf16 of one lane, CH in {2, 4, 8}.
template <int CH>
__device__ __forceinline__ void load_lane(const uint16_t* p, float (&x)[CH]) {
    uint32_t w[CH / 2];
    if constexpr (CH == 8) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else if constexpr (CH == 4) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        w[0] = u.x; w[1] = u.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
#pragma unroll
    for (int i = 0; i < CH / 2; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

template <int CH>
__device__ __forceinline__ void store_lane(uint16_t* p, const float (&x)[CH]) {
    uint32_t w[CH / 2];
#pragma unroll
    for (int i = 0; i < CH / 2; ++i)
        w[i] = static_cast<uint32_t>(bf_bits(x[2 * i])) | (static_cast<uint32_t>(bf_bits(x[2 * i + 1])) << 16);
    if constexpr (CH == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (CH == 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
}

// CH consecutive floats from shared memory, aligned as they are long up to 16 bytes.
template <int CH>
__device__ __forceinline__ void load_floats(const float* p, float (&x)[CH]) {
    if constexpr (CH >= 4) {
#pragma unroll
        for (int i = 0; i < CH; i += 4) {
            const float4 u = *reinterpret_cast<const float4*>(p + i);
            x[i] = u.x; x[i + 1] = u.y; x[i + 2] = u.z; x[i + 3] = u.w;
        }
    } else {
        const float2 u = *reinterpret_cast<const float2*>(p);
        x[0] = u.x; x[1] = u.y;
    }
}

// Quantises the row a warp holds (lane l: elements [l CH, l CH + CH)) in groups of `group`
// elements = group / CH lanes and writes codes, scales and biases.
//   edge e: the group's extreme of larger magnitude (the minimum only when strictly larger),
//   code of zero z = rint(e L / (max - min)) up to sign, scale s = e / z, bias b = e,
// each correctly rounded, so that a symmetric group's tie (e L / (max - min) = L / 2) goes to
// the even z on every path.  s and b are rounded to bf16, their stored form, BEFORE the codes
// are taken from them: with codes from the unrounded scale the 2^-9 of the scale would cost up
// to half a step at code 255.  Where (max - min) / L is under 1e-7 the step is 1e-7.
// A group with an element of kLargest or more, whose e L or max - min could pass fp32's range, is taken down
// by 2^-64 first and its scale and bias up again: powers of two, which change no rounding.  (Looking for such groups
// costs 0.5 us of 70 where 4102 rows of 32 heads are written in 4 bits and read back.)
constexpr float kLargest = 6.6461399789245794e35f;  // 2^119

template <int CH>
__device__ __forceinline__ void quantise_row(float (&x)[CH], int lane, int bits, int group, uint8_t* codes,
                                             uint16_t* scales, uint16_t* biases) {
    const float top = bits == 8 ? 255.f : 15.f;
    const int width = group / CH;  // lanes of a group, a power of two
    float lo = x[0], hi = x[0];
    bool small = true;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        small = small && fabsf(x[i]) < kLargest;
    }
    const uint32_t large = __ballot_sync(0xffffffffu, !small);
    for (int o = 1; o < width; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const uint32_t members = (width == 32 ? 0xffffffffu : (1u << width) - 1u) << (lane & ~(width - 1));
    bool bad = false;
    float up = 1.f, least = 1e-7f;
    if (large) {  // of the row, so seldom
        bool finite = true;
#pragma unroll
        for (int i = 0; i < CH; ++i) finite = finite && fabsf(x[i]) < INFINITY;
        bad = (__ballot_sync(0xffffffffu, !finite) & members) != 0;
        if (large & members) {
            const float down = 5.421010862427522e-20f;  // 2^-64
            up = 18446744073709551616.f;
            least *= down;
            lo *= down;
            hi *= down;
#pragma unroll
            for (int i = 0; i < CH; ++i) x[i] *= down;
        }
    }
    const bool low = fabsf(lo) > fabsf(hi);
    const float edge = low ? lo : hi, sign = low ? 1.f : -1.f, span = hi - lo;
    const bool tiny = span / top < least;
    const float z = sign * rintf(tiny ? edge / least : edge * top / span);
    float s = z != 0.f ? edge / z : sign * fmaxf(span / top, least);
    float b = z != 0.f ? edge : 0.f;
    if (bad) s = b = __int_as_float(0x7fc00000);
    uint16_t sb = bf_bits(s), bb = bf_bits(b);
    const float sr = __uint_as_float(static_cast<uint32_t>(sb) << 16), br = __uint_as_float(static_cast<uint32_t>(bb) << 16);
    if (large) {
        sb = bf_bits(sr * up);
        bb = bf_bits(br * up);
    }
    if ((lane & (width - 1)) == 0) {
        scales[lane / width] = sb;
        biases[lane / width] = bb;
    }
    // Codes are rint((x - b) / s) of the correctly rounded quotient.  The product with 1 / s is within 255 (2^-24 + 2^-24 +
    // 2^-24) = 4.6e-5 of it where it matters (further out both are clamped), so wherever it keeps 1e-4 from a tie it
    // rounds to the same code; a lane with an element nearer, or with a scale whose reciprocal could leave fp32's
    // normal range, divides.  (4102 rows x 32 heads in 4 bits, with the read-back: 91 us against 96.)
    const float inverse = 1.f / sr;
    bool divide = !(fabsf(sr) > 1e-30f && fabsf(sr) < 1e30f);
    float n[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const float t = (x[i] - br) * inverse;
        n[i] = rintf(t);
        divide = divide || !(fabsf(t - n[i]) < 0.4999f);
    }
    if (divide && !bad) {
#pragma unroll
        for (int i = 0; i < CH; ++i) n[i] = rintf((x[i] - br) / sr);
    }
    uint32_t c[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) c[i] = bad ? 0u : static_cast<uint32_t>(fminf(fmaxf(n[i], 0.f), top));
    if (bits == 8) {
        uint8_t* p = codes + lane * CH;
        if constexpr (CH == 8)
            *reinterpret_cast<uint2*>(p) = make_uint2(c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24,
                                                      c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24);
        else if constexpr (CH == 4) *reinterpret_cast<uint32_t*>(p) = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
        else *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(c[0] | c[1] << 8);
    } else {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < CH; ++i) w |= c[i] << (4 * i);
        uint8_t* p = codes + lane * CH / 2;
        if constexpr (CH == 8) *reinterpret_cast<uint32_t*>(p) = w;
        else if constexpr (CH == 4) *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w);
        else *p = static_cast<uint8_t>(w);
    }
}

// Writes one row that a warp holds to the cache in its format.
template <int CH>
__device__ __forceinline__ void store_cache_row(const View& cache, bool is_v, int64_t cr, int lane, float (&x)[CH]) {
    constexpr int d = CH * 32;
    uint8_t* base = (is_v ? cache.v : cache.k) + cr * (d * cache.bits / 8);
    if (cache.bits == 16) {
        store_lane<CH>(reinterpret_cast<uint16_t*>(base) + lane * CH, x);
    } else {
        const int64_t g = cr * (d / cache.group);
        quantise_row<CH>(x, lane, cache.bits, cache.group, base, (is_v ? cache.vs : cache.ks) + g,
                         (is_v ? cache.vb : cache.kb) + g);
    }
}

// Attention prep of a batch.  A CTA takes `rows_per` rows and `slots_per` head slots of each (slot < hq a q
// head, < hq + hkv a k head, else a v head), a warp one head at a time.  Lane l holds elements
// [l CH, l CH + CH) of the head, so every load and store of a row is one coalesced access and a group of
// the quantisation is a run of lanes.  Rotary: element i < rot / 2 pairs with i + rot / 2, which a whole
// number of lanes further on holds (rot / 2 is a multiple of 32); the rows' cosines and sines are made
// once per CTA and shared by its heads.  The angle is kept as a fraction of a turn in 64-bit fixed point:
// position times the frequency's fraction wraps as the angle does, so far positions lose little: the frequency, from
// 64-bit floating point, is off by up to 2^-54 of a turn a position, and the angle's rounding to fp32 adds 2^-26 of a turn
// (a float product is off by 2^-24 of the angle, 0.06 rad at a million).  The normalised k stays in 32 bits up
// to its one rounding, the quantisation.
constexpr int kPrepThreads = 256, kPrepRows = 2;

template <int CH>
__global__ void __launch_bounds__(kPrepThreads) attn_prep_batch_kernel(
    const uint16_t* qkv, long long ld, const uint16_t* __restrict__ q_norm, const uint16_t* __restrict__ k_norm,
    uint16_t* q_out, long long ld_q, View cache, const int32_t* __restrict__ lengths, int tokens, int hq, int rot,
    int position0, float eps, float theta, const int32_t* __restrict__ parents, int rows_per, int slots_per) {
    constexpr int d = CH * 32;
    __shared__ unsigned long long s_turn[d / 2];  // turns per position of pair i, 0.64 fixed point
    __shared__ __align__(16) float s_cos[kPrepRows][d / 2], s_sin[kPrepRows][d / 2];
    __shared__ int s_start[kPrepRows];            // first cache row of the row's block, -1: takes no part
    __shared__ int s_seq[kPrepRows];
    const int half = rot / 2;
    for (int i = threadIdx.x; i < half; i += kPrepThreads) {
        const double turns = exp2(-2.0 * i / rot * log2(static_cast<double>(theta))) * 0.15915494309189533577;
        s_turn[i] = static_cast<unsigned long long>((turns - floor(turns)) * 18446744073709551616.0);
    }
    pdl_wait();
    pdl_launch_dependents();
    const int r0 = blockIdx.x * rows_per, rows = min(rows_per, cache.sequences * tokens - r0);
    if (threadIdx.x < rows) {
        s_seq[threadIdx.x] = (r0 + threadIdx.x) / tokens;
        s_start[threadIdx.x] = block_start(lengths, s_seq[threadIdx.x], tokens, cache.max_len);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * half; i += kPrepThreads) {
        const int k = i / half, e = i - k * half, seq = s_seq[k], t = r0 + k - seq * tokens;
        const int depth = parents ? tree_walk(parents + (size_t)seq * tokens, t).depth : t;
        const unsigned long long a = s_turn[e] * static_cast<unsigned long long>((long long)position0 + s_start[k] + depth);
        sincospif(static_cast<float>(static_cast<int>(a >> 32)) * 4.656612873077392578125e-10f, &s_sin[k][e], &s_cos[k][e]);
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, hkv = cache.hkv, pair_lanes = half / CH;
    const int slot0 = blockIdx.y * slots_per, slots = min(slots_per, hq + 2 * hkv - slot0);
    const bool first = lane < pair_lanes, second = lane >= pair_lanes && lane < 2 * pair_lanes;
    const int other = first ? lane + pair_lanes : second ? lane - pair_lanes : lane;
    for (int it = threadIdx.x >> 5; it < rows * slots; it += kPrepThreads / 32) {
        const int k = it / slots, slot = slot0 + it - k * slots, start = s_start[k];
        if (start < 0) continue;
        const int r = r0 + k, seq = s_seq[k], t = r - seq * tokens;
        const bool is_v = slot >= hq + hkv, is_q = slot < hq;
        float x[CH];
        load_lane<CH>(qkv + (size_t)r * ld + (size_t)(is_q ? slot : hq + slot) * d + lane * CH, x);
        if (!is_v) {
            float w[CH];
            load_lane<CH>((is_q ? q_norm : k_norm) + lane * CH, w);
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < CH; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float rs = rsqrtf(ss / d + eps);
#pragma unroll
            for (int i = 0; i < CH; ++i) x[i] = x[i] * rs * w[i];
            if (rot > 0) {
                const int e = (second ? lane - pair_lanes : first ? lane : 0) * CH;
                float cs[CH], sn[CH];
                load_floats<CH>(&s_cos[k][e], cs);
                load_floats<CH>(&s_sin[k][e], sn);
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    const float y = __shfl_sync(0xffffffffu, x[i], other);
                    if (first) x[i] = x[i] * cs[i] - y * sn[i];
                    else if (second) x[i] = x[i] * cs[i] + y * sn[i];
                }
            }
        }
        if (is_q)
            store_lane<CH>(q_out + (size_t)r * ld_q + (size_t)slot * d + lane * CH, x);
        else
            store_cache_row<CH>(cache, is_v, row_index(cache, seq, is_v ? slot - hq - hkv : slot - hq, start + t), lane, x);
    }
}

// Eight consecutive elements of a cache row as bf16, e0 a multiple of 8.
__device__ __forceinline__ uint4 read8(const uint8_t* codes, const uint16_t* scales, const uint16_t* biases, int64_t row,
                                       int d, int bits, int group, int e0) {
    const uint8_t* p = codes + row * (d * bits / 8) + e0 * bits / 8;
    if (bits == 16) return *reinterpret_cast<const uint4*>(p);
    const int64_t g = row * (d / group) + e0 / group;
    const float s = bf16_bits_to_float(scales[g]), b = bf16_bits_to_float(biases[g]);
    uint32_t out[4];
    if (bits == 8) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = (i < 2 ? u.x : u.y) >> (16 * (i & 1));
            out[i] = bf_bits(fmaf(s, static_cast<float>(w & 255u), b)) |
                     static_cast<uint32_t>(bf_bits(fmaf(s, static_cast<float>((w >> 8) & 255u), b))) << 16;
        }
    } else {
        const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = u >> (8 * i);
            out[i] = bf_bits(fmaf(s, static_cast<float>(w & 15u), b)) |
                     static_cast<uint32_t>(bf_bits(fmaf(s, static_cast<float>((w >> 4) & 15u), b))) << 16;
        }
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}

// Read-back of cache rows: one thread per eight elements, k and v alike.
__global__ void __launch_bounds__(256) kv_read_kernel(View cache, const int32_t* __restrict__ starts, int rows,
                                                      uint16_t* __restrict__ k, uint16_t* __restrict__ v) {
    pdl_wait();
    pdl_launch_dependents();
    const int per_row = cache.d / 8;  // a power of two
    const long long n = (long long)cache.sequences * cache.hkv * rows * per_row;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        // 2^32 rows of at least 128 bytes of output are more than a GPU has
        const uint32_t line = static_cast<uint32_t>(i >> (__ffs(per_row) - 1)), of_head = line / rows;
        const int e0 = static_cast<int>(i & (per_row - 1)) * 8, row = static_cast<int>(line - of_head * rows);
        const int seq = static_cast<int>(of_head / cache.hkv), head = static_cast<int>(of_head - seq * cache.hkv);
        const int start = starts ? block_start(starts, seq, rows, cache.max_len) : 0;
        if (start < 0) continue;
        const int64_t cr = row_index(cache, seq, head, start + row);
        if (k) reinterpret_cast<uint4*>(k)[i] = read8(cache.k, cache.ks, cache.kb, cr, cache.d, cache.bits, cache.group, e0);
        if (v) reinterpret_cast<uint4*>(v)[i] = read8(cache.v, cache.vs, cache.vb, cr, cache.d, cache.bits, cache.group, e0);
    }
}

// Rows taken as they are, one warp per (sequence, kv head, row, k or v).
template <int CH>
__global__ void __launch_bounds__(256) kv_write_kernel(View cache, const int32_t* __restrict__ starts, int rows,
                                                       const uint16_t* __restrict__ k, const uint16_t* __restrict__ v) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const long long n = (long long)cache.sequences * cache.hkv * rows;
    for (long long it = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); it < 2 * n; it += (long long)gridDim.x * 8) {
        const bool is_v = it >= n;
        const long long i = is_v ? it - n : it;
        const int row = static_cast<int>(i % rows), head = static_cast<int>(i / rows % cache.hkv);
        const int seq = static_cast<int>(i / rows / cache.hkv);
        const int start = starts ? block_start(starts, seq, rows, cache.max_len) : 0;
        if (start < 0) continue;
        float x[CH];
        load_lane<CH>((is_v ? v : k) + i * (CH * 32) + lane * CH, x);
        store_cache_row<CH>(cache, is_v, row_index(cache, seq, head, start + row), lane, x);
    }
}

// Rows of an accepted tree path to the block's front; grid (kv head, sequence, k or v).  All
// rows are staged in shared memory before any is written, so overlapping moves are safe.
__global__ void __launch_bounds__(256) kv_compact_batch_kernel(View cache, const int32_t* __restrict__ lengths,
                                                               const int32_t* __restrict__ rows,
                                                               const int32_t* __restrict__ counts, int stride) {
    __shared__ uint4 s_row[kMaxTreeRows * 32];                       // up to 512 bytes a row
    __shared__ uint16_t s_group[2][kMaxTreeRows * 8];                // up to 8 groups a row
    pdl_wait();
    pdl_launch_dependents();
    const int head = blockIdx.x, seq = blockIdx.y;
    const int n = lengths[seq], keep = counts[seq];
    if (n < 0) return;
    const int32_t* r = rows + (size_t)seq * stride;
    bool ok = keep >= 0 && keep <= stride;
    for (int i = 0; ok && i < keep; ++i) ok = r[i] >= 0 && r[i] < kMaxTreeRows && r[i] < cache.max_len - n;
    if (!ok || keep > cache.max_len - n) {
        if (threadIdx.x == 0) atomicOr(&g_device_error, DFLASH_DEVERR_POSITION);
        return;
    }
    const int words = cache.d * cache.bits / 128, groups = cache.bits == 16 ? 0 : cache.d / cache.group;
    const int64_t base = row_index(cache, seq, head, n);
    uint4* data = reinterpret_cast<uint4*>(blockIdx.z ? cache.v : cache.k) + base * words;
    uint16_t* sc = (blockIdx.z ? cache.vs : cache.ks) + base * groups;
    uint16_t* bi = (blockIdx.z ? cache.vb : cache.kb) + base * groups;
    for (int i = threadIdx.x; i < keep * words; i += blockDim.x) s_row[i] = data[(int64_t)r[i / words] * words + i % words];
    for (int i = threadIdx.x; i < keep * groups; i += blockDim.x) {
        s_group[0][i] = sc[(int64_t)r[i / groups] * groups + i % groups];
        s_group[1][i] = bi[(int64_t)r[i / groups] * groups + i % groups];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < keep * words; i += blockDim.x) data[i] = s_row[i];
    for (int i = threadIdx.x; i < keep * groups; i += blockDim.x) {
        sc[i] = s_group[0][i];
        bi[i] = s_group[1][i];
    }
}

inline bool stride_ok(const void* p, long long ld, long long need) { return aligned16(p) && ld >= need && ld % 8 == 0; }

}  // namespace kv
}  // namespace dflash

extern "C" int dflash_stack_attn_prep_batch(const dflash_bf16* qkv, long long ld, const dflash_bf16* q_norm,
                                            const dflash_bf16* k_norm, dflash_bf16* q_out, long long ld_q,
                                            const dflash_kv_cache* cache, const int32_t* lengths, int tokens, int hq,
                                            int rot, int position0, float eps, float theta, const int32_t* parents,
                                            dflash_stream_t stream) {
    using namespace dflash;
    const char* who = "dflash_stack_attn_prep_batch";
    const int st = kv::check_cache(cache, who);
    if (st != DFLASH_OK) return st;
    const int d = cache->head_dim, hkv = cache->kv_heads;
    if (!qkv || !q_norm || !k_norm || !q_out || !lengths || tokens < 1 || tokens > cache->max_len || hq < 1 ||
        position0 < 0 || !(theta > 0.f) || (parents && tokens > kMaxTreeRows))
        return fail(DFLASH_ERR_INVALID_ARGUMENT, "%s: bad arguments", who);
    if (hq > 65535 || (long long)cache->sequences * tokens > 0x7fffffffll / (hq + 2 * hkv) ||
        (long long)position0 + cache->max_len > 0x7fffffffll)
        return fail(DFLASH_ERR_UNSUPPORTED, "%s: too many rows, heads or positions", who);
    if (rot < 0 || rot > d || rot % 64)
        return fail(DFLASH_ERR_UNSUPPORTED, "%s: rotary dims %d: a multiple of 64 up to %d", who, rot, d);
    if (ld < (2ll * hq + 2ll * hkv) * d || ld_q < (long long)hq * d)
        return fail(DFLASH_ERR_INVALID_ARGUMENT, "%s: row strides too small", who);
    if (!kv::stride_ok(qkv, ld, 1) || !kv::stride_ok(q_out, ld_q, 1) || !aligned16(q_norm) || !aligned16(k_norm))
        return fail(DFLASH_ERR_MISALIGNED, "%s: qkv, q_out, their row strides and the norm weights must be 16-byte "
                    "aligned", who);
    int dev = 0;
    DFLASH_CUDA_TRY(cudaGetDevice(&dev));
    // many rows: two of them and all their heads per CTA, whose cosines are then made once; few: a row and eight
    // heads per CTA, a head per warp.  With the read-back, 8 rows x 32 heads: 6.4 us as few, 15 as many; 4102 rows:
    // 94 us as few, 70 as many (four rows per CTA 77, eight 91: too few warps hide the 1.3 us that a head takes)
    const long long rows = (long long)cache->sequences * tokens;
    const int slots = hq + 2 * hkv;
    const bool many = rows * slots >= 64ll * sm_count(dev);
    const int rows_per = many ? kv::kPrepRows : 1, slots_per = many ? slots : kv::kPrepThreads / 32;
    const dim3 grid(static_cast<unsigned>((rows + rows_per - 1) / rows_per), (slots + slots_per - 1) / slots_per),
        block(kv::kPrepThreads);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const kv::View c = kv::view_of(*cache);
    cudaError_t e;
    switch (d) {
        case 64: e = launch_chained(kv::attn_prep_batch_kernel<2>, grid, block, 0, s, 1, qkv, ld, q_norm, k_norm, q_out,
                                    ld_q, c, lengths, tokens, hq, rot, position0, eps, theta, parents, rows_per, slots_per); break;
        case 128: e = launch_chained(kv::attn_prep_batch_kernel<4>, grid, block, 0, s, 1, qkv, ld, q_norm, k_norm, q_out,
                                     ld_q, c, lengths, tokens, hq, rot, position0, eps, theta, parents, rows_per, slots_per); break;
        default: e = launch_chained(kv::attn_prep_batch_kernel<8>, grid, block, 0, s, 1, qkv, ld, q_norm, k_norm, q_out,
                                    ld_q, c, lengths, tokens, hq, rot, position0, eps, theta, parents, rows_per, slots_per);
    }
    DFLASH_CUDA_TRY(e);
    return DFLASH_OK;
}

extern "C" int dflash_stack_kv_read(const dflash_kv_cache* cache, const int32_t* starts, int rows, dflash_bf16* k,
                                    dflash_bf16* v, dflash_stream_t stream) {
    using namespace dflash;
    const int st = kv::check_cache(cache, "dflash_stack_kv_read");
    if (st != DFLASH_OK) return st;
    if ((!k && !v) || rows < 1 || rows > cache->max_len)
        return fail(DFLASH_ERR_INVALID_ARGUMENT, "dflash_stack_kv_read: bad arguments");
    if ((k && !aligned16(k)) || (v && !aligned16(v)))
        return fail(DFLASH_ERR_MISALIGNED, "dflash_stack_kv_read: k and v must be 16-byte aligned");
    int dev = 0;
    DFLASH_CUDA_TRY(cudaGetDevice(&dev));
    const long long n = (long long)cache->sequences * cache->kv_heads * rows * (cache->head_dim / 8);
    const long long blocks = (n + 255) / 256, most = 16ll * sm_count(dev);
    DFLASH_CUDA_TRY(launch_chained(kv::kv_read_kernel, dim3(static_cast<unsigned>(blocks < most ? blocks : most)), dim3(256),
                                   0, reinterpret_cast<cudaStream_t>(stream), 1, kv::view_of(*cache), starts, rows, k, v));
    return DFLASH_OK;
}

extern "C" int dflash_stack_kv_write(const dflash_kv_cache* cache, const int32_t* starts, int rows, const dflash_bf16* k,
                                     const dflash_bf16* v, dflash_stream_t stream) {
    using namespace dflash;
    const int st = kv::check_cache(cache, "dflash_stack_kv_write");
    if (st != DFLASH_OK) return st;
    if (!k || !v || rows < 1 || rows > cache->max_len)
        return fail(DFLASH_ERR_INVALID_ARGUMENT, "dflash_stack_kv_write: bad arguments");
    if (!aligned16(k) || !aligned16(v))
        return fail(DFLASH_ERR_MISALIGNED, "dflash_stack_kv_write: k and v must be 16-byte aligned");
    int dev = 0;
    DFLASH_CUDA_TRY(cudaGetDevice(&dev));
    const long long blocks = (2ll * cache->sequences * cache->kv_heads * rows + 7) / 8, most = 8ll * sm_count(dev);
    const dim3 grid(static_cast<unsigned>(blocks < most ? blocks : most)), block(256);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const kv::View c = kv::view_of(*cache);
    cudaError_t e;
    switch (cache->head_dim) {
        case 64: e = launch_chained(kv::kv_write_kernel<2>, grid, block, 0, s, 1, c, starts, rows, k, v); break;
        case 128: e = launch_chained(kv::kv_write_kernel<4>, grid, block, 0, s, 1, c, starts, rows, k, v); break;
        default: e = launch_chained(kv::kv_write_kernel<8>, grid, block, 0, s, 1, c, starts, rows, k, v);
    }
    DFLASH_CUDA_TRY(e);
    return DFLASH_OK;
}

extern "C" int dflash_stack_kv_compact_batch(const dflash_kv_cache* cache, const int32_t* lengths, const int32_t* rows,
                                             const int32_t* counts, int stride, dflash_stream_t stream) {
    using namespace dflash;
    const int st = kv::check_cache(cache, "dflash_stack_kv_compact_batch");
    if (st != DFLASH_OK) return st;
    if (!lengths || !rows || !counts || stride < 1 || stride > kMaxTreeRows)
        return fail(DFLASH_ERR_INVALID_ARGUMENT, "dflash_stack_kv_compact_batch: bad arguments (1 to %d rows)", kMaxTreeRows);
    DFLASH_CUDA_TRY(launch_chained(kv::kv_compact_batch_kernel, dim3(cache->kv_heads, cache->sequences, 2), dim3(256), 0,
                                   reinterpret_cast<cudaStream_t>(stream), 1, kv::view_of(*cache), lengths, rows, counts,
                                   stride));
    return DFLASH_OK;
}
