// Decode attention of a batch of sequences over caches of 16, 8 or 4 bits, with an optional
// prefix that all of them share (include/dflash_batch.h).
//
// Work is cut into tiles of kKeys = 128 keys of one kv head against a block of up to kRows = 128
// query rows: the S T G rows of the whole batch for the prefix, the T G rows of one sequence for
// its own cache.  The list of all tiles (prefix first; its length follows from `lengths` on the
// device) is cut into equal runs, one per CTA, so any mix of lengths loads the SMs evenly; the
// part of a run inside one (row block, kv head) leaves a partial (max, sum, p V) in the workspace
// and a second kernel joins them.
//
// A tile is two products on the tensor cores, keys and head dimensions on the 128-row side, query
// rows on the column side:
//   S^T [128 keys x rows]  = K [128 x d] Q^T           K as it lies in the cache
//   O^T [d x rows]        += V^T [d x 128] P^T         V as it lies in the cache, read transposed
// so few rows waste nothing (a product costs as long as reading its 128-row operand from shared
// memory up to 64 rows), no operand is transposed by a thread, and a thread that reads S^T owns
// one key: its mask and its scale factors are its own registers.  Q, K, V and P are bf16 over bf16
// caches.  Over quantised caches they are fp16, whose 11 bits lose little to the codes' 8: every
// key's values (and every query row) are first scaled by a power of two into fp16's upper range,
// undone in S^T for K and Q, and for V folded into P's exponent and the sum's weights.
//
// Roles: warps 0-7 softmax (two per TMEM lane quarter, half of the columns each), 8-15 producers
// (cache rows to swizzled shared memory boxes of 128 keys x 64 elements, in a ring), warp 16 issues
// the products.  The running maximum is only raised when a score passes it by kLazy (in powers
// of two), so the accumulators are rarely rescaled.
#include "common.cuh"
#include "dflash_batch.h"
#include "tcgen05.cuh"

namespace dflash {
namespace attn {

constexpr int kKeys = 128;
constexpr int kRows = 128;
constexpr int kBox = kKeys * 128;          // bytes of a ring slot: 128 keys x 64 elements of 16 bits
constexpr int kSoftmaxWarps = 8, kProducerWarps = 8;
constexpr int kThreads = 32 * (kSoftmaxWarps + kProducerWarps + 1);
constexpr int kMaxCtas = 160;              // partials are sized for this many CTAs
constexpr int kMaxSlots = 10;
constexpr int kScaleDepth = 4;             // tiles whose key factors may be alive at once
constexpr int kPoison = 16;                // units whose poison flags may be alive at once
constexpr float kLazy = 4.f;               // a maximum moves when a score passes it by 2^4 ...
constexpr float kLift = 8.f;               // ... and P is 2^8 p, up to 2^12: small weights stay normal in fp16
constexpr int kTop = 12;                   // fp16 operands are scaled to 2^12 .. 2^13
constexpr uint32_t kTmemColumns = 512;
constexpr int kSmemLimit = 232448 - 1024;

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
    // sizes that follow from the above
    int G, blocks_p, blocks_o;   // row blocks of the prefix and of one sequence
    int rows_o;                  // rows of a block of one sequence, at most
    int nr;                      // columns of the products' buffers: 64 or kRows
    int slots;                   // ring slots
    // workspace: partials of the prefix, then of the sequences
    int32_t* first;              // [segments] first and last CTA of each (row block, kv head)
    int32_t* last;
    int32_t* poison;             // [partials]
    float2* ml;                  // [partials][rows] (max in powers of two, sum)
    float* o;                    // [partials][rows][d]
};

// Partials of the prefix are (segment + CTA), of the sequences behind them; a run of tiles crosses
// a segment or a CTA border at each step, so segment + CTA is its own for every piece.
__host__ __device__ inline long long segments_p(const Args& a) { return (long long)a.blocks_p * a.cache.hkv; }
__host__ __device__ inline long long segments_o(const Args& a) {
    return (long long)a.cache.sequences * a.blocks_o * a.cache.hkv;
}
__host__ __device__ inline long long partials_p(const Args& a) { return a.blocks_p ? segments_p(a) + kMaxCtas : 0; }
__host__ __device__ inline long long partials_o(const Args& a) { return segments_o(a) + kMaxCtas; }
// Index of row 0 of a partial in ml (and, times d, in o).
__device__ __forceinline__ long long partial_row(const Args& a, bool prefix, long long segment, int cta) {
    return prefix ? (segment + cta) * kRows : partials_p(a) * kRows + (segment + cta) * a.rows_o;
}
__device__ __forceinline__ long long partial_index(const Args& a, bool prefix, long long segment, int cta) {
    return prefix ? segment + cta : partials_p(a) + segment + cta;
}

// Shared memory behind the ring, Q and P: offsets in bytes.
struct Layout {
    uint32_t q, p, scale_k, scale_v, key_k, key_v, key_w, row, part, bars, misc, total;
};
__host__ __device__ inline Layout layout(int d, int nr, int slots, int groups) {
    Layout l;
    uint32_t at = slots * kBox;
    l.q = at;             at += nr * d * 2;
    l.p = at;             at += kKeys * nr * 2;
    l.scale_k = at;       at += kKeys * groups * 4;
    l.scale_v = at;       at += 2 * kKeys * groups * 4;
    l.key_k = at;         at += groups ? kScaleDepth * kKeys * 4 : 0;
    l.key_v = at;         at += groups ? kScaleDepth * kKeys * 4 : 0;
    l.key_w = at;         at += groups ? kScaleDepth * kKeys * 2 : 0;
    l.row = at;           at += 6 * kRows * 4;
    l.part = at;          at += 4 * kRows * 4;
    l.bars = at;          at += 8 * (2 * kMaxSlots + 2 + 1 + 1 + 1 + 2 * kScaleDepth + 1);
    l.misc = at;          at += 4 * (kPoison + 8 + 40);
    l.total = at;
    return l;
}

// ---------------------------------------------------------------- units of a CTA's run
// A unit: consecutive tiles of one (row block, kv head).
struct Unit {
    bool prefix;
    int head, seq, block;   // seq: sequence (own) ; block: row block
    long long segment;
    int t0, n;              // tiles t0 .. t0 + n - 1 of the segment
    int tiles;              // tiles of the segment
    int rows;               // query rows
    int len;                // own: cached tokens before the block; prefix: prefix_len
    int keys;               // keys that some row sees
};

__device__ __forceinline__ int own_keys(const Args& a, int len, int block) {
    const int last = min(a.tokens * a.G, (block + 1) * kRows) - 1;
    return a.parents ? len + a.tokens : len + last / a.G + 1;
}
__device__ __forceinline__ int live_length(const Args& a, int seq) {
    const int n = a.lengths[seq];
    return n > a.cache.max_len - a.tokens ? -1 : n;
}
__device__ __forceinline__ int entry_tiles(const Args& a, int e) {
    const int len = live_length(a, e / a.blocks_o);
    return len < 0 ? 0 : (own_keys(a, len, e % a.blocks_o) + kKeys - 1) / kKeys;
}

struct Walker {
    int w, w1;          // next tile and end of the run
    int entry, off;     // own region: current (sequence, row block) and its first tile
    __device__ __forceinline__ bool next(const Args& a, Unit& u) {
        if (w >= w1) return false;
        const int tiles_p = (a.prefix_len + kKeys - 1) / kKeys, prefix_end = tiles_p * a.blocks_p * a.cache.hkv;
        if (w < prefix_end) {
            const int s = w / tiles_p;
            u.prefix = true;
            u.segment = s;
            u.block = s / a.cache.hkv;
            u.head = s % a.cache.hkv;
            u.seq = 0;
            u.tiles = tiles_p;
            u.t0 = w - s * tiles_p;
            u.rows = min(kRows, a.cache.sequences * a.tokens * a.G - u.block * kRows);
            u.len = u.keys = a.prefix_len;
        } else {
            int tiles = entry_tiles(a, entry);
            while (w >= off + tiles * a.cache.hkv) {
                off += tiles * a.cache.hkv;
                tiles = entry_tiles(a, ++entry);
            }
            const int rel = w - off;
            u.prefix = false;
            u.head = rel / tiles;
            u.seq = entry / a.blocks_o;
            u.block = entry % a.blocks_o;
            u.segment = (long long)entry * a.cache.hkv + u.head;
            u.tiles = tiles;
            u.t0 = rel - u.head * tiles;
            u.rows = min(kRows, a.tokens * a.G - u.block * kRows);
            u.len = a.lengths[u.seq];
            u.keys = own_keys(a, u.len, u.block);
        }
        u.n = min(u.tiles - u.t0, w1 - w);
        w += u.n;
        return true;
    }
};

// ---------------------------------------------------------------- small helpers
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float warp_max(float x) {  // NaN counts as nothing
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t fma_h2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t sub_h2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool fill) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(fill ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// bar.red.or over `threads` threads of barrier `id`.
__device__ __forceinline__ bool bar_any(int id, int threads, bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, %2, %3, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(static_cast<uint32_t>(v)), "r"(id), "r"(threads)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }  // 2^e, e in -126 .. 127
// Exponent of |a| for the scaling: 0 for zero, infinity and NaN.
__device__ __forceinline__ int exponent(float a) {
    const int e = (__float_as_int(a) >> 23) & 255;
    return e == 0 || e == 255 ? 0 : e - 127;
}

// Within each eight elements the 4-bit unpack leaves this order (pairs i, i + 4).
template <int BITS>
__device__ __forceinline__ int order(int i) {
    return BITS == 4 ? (i >> 1) + 4 * (i & 1) : i;
}

// ---------------------------------------------------------------- the kernel
template <int BITS, int D>
struct Kernel {
    static constexpr bool kQuant = BITS != 16;
    static constexpr int NB = D / 64;                  // boxes of a K or V tile
    static constexpr int MB = D > 64 ? D / 128 : 1;    // 128-lane blocks of O^T (half used when d is 64)
    static constexpr int kLoads = kQuant ? NB * BITS / 4 : 1;  // 16-byte loads of codes a producer thread makes per tile

    struct Shared {
        uint32_t base;  // shared address of the ring
        Layout l;
        uint64_t *full, *empty, *s_full, *p_full, *pv_done, *q_full, *sc_full, *sc_empty;
        int* poison;
        int* misc;  // 0 abort, 1 tmem, 2 run start, 3 run end, 4 entry, 5 off
        volatile int* abort;
        float *thr, *mm, *qs, *corr, *m;
        int* rowinfo;  // chain: the row's token; tree: its path mask
        float* part;
    };

    __device__ static __forceinline__ void wait(const Shared& s, uint64_t* bar, uint32_t parity) {
        mbar_wait_bounded(bar, parity, s.abort, DFLASH_DEVERR_ATTN_PIPELINE);
    }

    // ------------------------------------------------------------ producers
    struct Tile {            // where a tile's rows lie
        const kv::View* c;
        int64_t row0;
        int valid;           // rows that exist and that some query row sees
        int suspect;         // rows from here on are hidden from some query row
        int poison;          // flag of the unit
    };
    struct TileWalk {
        Walker w;
        Unit u;
        int i, unit;
        __device__ __forceinline__ bool next(const Args& a, Tile& t, bool& first) {
            first = false;
            if (i == u.n) {
                if (!w.next(a, u)) return false;
                i = 0;
                ++unit;
                first = true;
            }
            const int tile = u.t0 + i++;
            t.c = u.prefix ? &a.prefix : &a.cache;
            t.row0 = kv::row_index(*t.c, u.seq, u.head, tile * kKeys);
            t.valid = min(kKeys, u.keys - tile * kKeys);
            t.suspect = u.prefix ? kKeys : max(0, u.len - tile * kKeys);
            t.poison = unit & (kPoison - 1);
            return true;
        }
    };

    struct Ring {
        int slot;
        uint32_t phase;
        __device__ __forceinline__ void step(int slots) {
            if (++slot == slots) {
                slot = 0;
                phase ^= 1;
            }
        }
    };

    // A non-finite element of a row that some query row does not see would reach it as 0 * inf: it
    // is taken out of the operand and the unit's flag raised, for the join to put it back where it
    // is seen.  v holds eight 16-bit elements.
    __device__ static __forceinline__ void clean(uint4& v, int* flag) {
        constexpr uint32_t kExp = kQuant ? 0x7c00u : 0x7f80u;
        uint32_t* w = &v.x;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if ((w[i] & kExp) == kExp) { w[i] &= 0xffff0000u; bad = true; }
            if ((w[i] & (kExp << 16)) == (kExp << 16)) { w[i] &= 0x0000ffffu; bad = true; }
        }
        if (bad) *flag = 1;
    }

    __device__ static __forceinline__ void signal_full(const Shared& s, int slot) {
        fence_proxy_async_shared();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&s.full[slot]);
    }

    // bf16 caches: cp.async straight into the swizzled boxes, up to kLag boxes in flight.
    static constexpr int kLag = 5;

    __device__ static void produce_bf16(const Args& a, const Shared& s, Walker w0) {
        const int pt = threadIdx.x - 32 * kSoftmaxWarps;
        Ring ring{0, 0};
        int done_slot = 0, pending = 0;
        // what to look at in the boxes in flight (a queue of kLag)
        int q_from[kLag] = {}, q_flag[kLag] = {};
        const auto retire = [&]() {  // the oldest box in flight is complete
            if (q_from[0] < kKeys) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int key = (pt + 256 * u) >> 3, c = pt & 7;
                    if (key >= q_from[0]) {
                        const uint32_t addr = s.base + done_slot * kBox + key * 128 + ((c ^ (key & 7)) << 4);
                        uint4 v = lds128(addr);
                        clean(v, &s.poison[q_flag[0]]);
                        sts128(addr, v);
                    }
                }
            }
            signal_full(s, done_slot);
            if (++done_slot == a.slots) done_slot = 0;
#pragma unroll
            for (int i = 0; i + 1 < kLag; ++i) {
                q_from[i] = q_from[i + 1];
                q_flag[i] = q_flag[i + 1];
            }
            --pending;
        };
        const auto wait_oldest = [&]() {
            switch (pending) {
                case 1: cp_async_wait<0>(); break;
                case 2: cp_async_wait<1>(); break;
                case 3: cp_async_wait<2>(); break;
                case 4: cp_async_wait<3>(); break;
                default: cp_async_wait<4>(); break;
            }
            retire();
        };
        const auto box = [&](const Tile& t, bool is_v, int b) {
            if (pending == kLag) wait_oldest();
            const uint32_t parity = ring.phase ^ 1;
            while (pending > 0 && !mbar_try_wait(&s.empty[ring.slot], parity)) wait_oldest();
            wait(s, &s.empty[ring.slot], parity);
            const uint16_t* src = reinterpret_cast<const uint16_t*>(is_v ? t.c->v : t.c->k);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int key = (pt + 256 * u) >> 3, c = pt & 7;
                const bool live = key < t.valid;
                cp_async16(s.base + ring.slot * kBox + key * 128 + ((c ^ (key & 7)) << 4),
                           src + (t.row0 + (live ? key : 0)) * D + b * 64 + c * 8, live);
            }
            cp_async_commit();
#pragma unroll
            for (int i = 0; i < kLag; ++i)
                if (i == pending) {
                    q_from[i] = is_v && t.suspect < t.valid ? t.suspect : kKeys;
                    q_flag[i] = t.poison;
                }
            ++pending;
            ring.step(a.slots);
        };
        TileWalk tw{w0, Unit{}, 0, -1};
        tw.u.n = 0;
        Tile t, prev;
        bool first, have_prev = false;
        while (tw.next(a, t, first)) {
            if (first && have_prev) {  // the unit before ends with its last V
                for (int b = 0; b < NB; ++b) box(prev, true, b);
                have_prev = false;
            }
            for (int b = 0; b < NB; ++b) box(t, false, b);
            if (have_prev)
                for (int b = 0; b < NB; ++b) box(prev, true, b);
            prev = t;
            have_prev = true;
        }
        if (have_prev)
            for (int b = 0; b < NB; ++b) box(prev, true, b);
        while (pending > 0) wait_oldest();
    }

    // Quantised caches: codes to registers a tile ahead, unpacked to fp16 and stored swizzled.
    __device__ static __forceinline__ void load_codes(const Tile& t, bool is_v, int pt, uint4 (&r)[kLoads]) {
        const uint8_t* src = (is_v ? t.c->v : t.c->k) + t.row0 * (D * BITS / 8);
        constexpr int kPer = BITS / 2;  // 16-byte pieces of a key in a box
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int box = i / (BITS / 4), idx = pt + 256 * (i % (BITS / 4)), key = idx / kPer, piece = idx % kPer;
            r[i] = key < t.valid ? __ldcs(reinterpret_cast<const uint4*>(src + (size_t)key * (D * BITS / 8) + box * (8 * BITS) +
                                                                         piece * 16))
                                 : make_uint4(0, 0, 0, 0);
        }
    }
    // Scales and biases of one key, as raw bf16 pairs.
    struct Groups {
        uint32_t s[4], b[4];
    };
    __device__ static __forceinline__ void load_groups(const Tile& t, bool is_v, int key, int groups, Groups& g) {
        const uint16_t* ps = (is_v ? t.c->vs : t.c->ks) + (t.row0 + key) * groups;
        const uint16_t* pb = (is_v ? t.c->vb : t.c->kb) + (t.row0 + key) * groups;
#pragma unroll
        for (int i = 0; i < 4; ++i) g.s[i] = g.b[i] = 0;
        if (key >= t.valid) return;
        if (groups == 1) {
            g.s[0] = *ps;
            g.b[0] = *pb;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (2 * i < groups) {
                    g.s[i] = reinterpret_cast<const uint32_t*>(ps)[i];
                    g.b[i] = reinterpret_cast<const uint32_t*>(pb)[i];
                }
        }
    }
    // Largest magnitude that a key's groups can stand for.
    __device__ static __forceinline__ float largest(const Groups& g, int groups) {
        constexpr float kCodes = BITS == 8 ? 255.f : 15.f;
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < groups) {
                const float sc = __uint_as_float(i & 1 ? g.s[i / 2] & 0xffff0000u : g.s[i / 2] << 16);
                const float bi = __uint_as_float(i & 1 ? g.b[i / 2] & 0xffff0000u : g.b[i / 2] << 16);
                m = fmaxf(m, fmaxf(fabsf(bi), fabsf(fmaf(kCodes, sc, bi))));
            }
        return m;
    }
    __device__ static __forceinline__ void store_groups(uint32_t addr, const Groups& g, int groups, float f) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < groups) {
                const float sc = __uint_as_float(i & 1 ? g.s[i / 2] & 0xffff0000u : g.s[i / 2] << 16);
                const float bi = __uint_as_float(i & 1 ? g.b[i / 2] & 0xffff0000u : g.b[i / 2] << 16);
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr + 4 * i), "r"(pack2<false>(sc * f, bi * f)) : "memory");
            }
    }
    // Unpacks one 16-byte piece (32 or 16 elements of one key and group) into its 16-byte chunks of a box.
    __device__ static __forceinline__ void unpack(uint4 codes, uint32_t sb, uint32_t row_addr, int key, int piece, bool suspect,
                                                  int* flag) {
        const uint32_t s2 = __byte_perm(sb, 0, 0x1010), b2 = __byte_perm(sb, 0, 0x3232);
        const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
        constexpr uint32_t kMagic = 0x64006400u;  // fp16 1024 + code
        if constexpr (BITS == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint4 v;
                uint32_t* p = &v.x;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    p[j] = fma_h2(sub_h2((w[i] >> (4 * j)) & 0x000f000fu | kMagic, kMagic), s2, b2);
                if (suspect) clean(v, flag);
                sts128(row_addr + (((4 * piece + i) ^ (key & 7)) << 4), v);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint4 v;
                v.x = fma_h2(sub_h2(__byte_perm(w[2 * i], kMagic, 0x5150), kMagic), s2, b2);
                v.y = fma_h2(sub_h2(__byte_perm(w[2 * i], kMagic, 0x5352), kMagic), s2, b2);
                v.z = fma_h2(sub_h2(__byte_perm(w[2 * i + 1], kMagic, 0x5150), kMagic), s2, b2);
                v.w = fma_h2(sub_h2(__byte_perm(w[2 * i + 1], kMagic, 0x5352), kMagic), s2, b2);
                if (suspect) clean(v, flag);
                sts128(row_addr + (((2 * piece + i) ^ (key & 7)) << 4), v);
            }
        }
    }

    __device__ static void produce_quant(const Args& a, const Shared& s, Walker w0) {
        const int pt = threadIdx.x - 32 * kSoftmaxWarps, groups = D / a.cache.group;
        const int key_of = pt & (kKeys - 1);
        const bool does_v = pt >= kKeys;
        Ring ring{0, 0};
        const auto emit = [&](const Tile& t, bool is_v, const uint4 (&r)[kLoads], uint32_t table) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                wait(s, &s.empty[ring.slot], ring.phase ^ 1);
                const uint32_t box = s.base + ring.slot * kBox;
                constexpr int kPer = BITS / 2;
#pragma unroll
                for (int u = 0; u < BITS / 4; ++u) {
                    const int idx = pt + 256 * u, key = idx / kPer, piece = idx % kPer;
                    const int element = b * 64 + piece * (128 / BITS);
                    const uint32_t sb = lds32(table + (key * groups + element / a.cache.group) * 4);
                    unpack(r[b * (BITS / 4) + u], sb, box + key * 128, key, piece, is_v && key >= t.suspect && key < t.valid,
                           &s.poison[t.poison]);
                }
                signal_full(s, ring.slot);
                ring.step(a.slots);
            }
        };
        TileWalk tw{w0, Unit{}, 0, -1};
        tw.u.n = 0;
        Tile t, next, prev;
        bool first, next_first = false, more;
        uint4 kr[kLoads], vr[kLoads];
        Groups g;
        if (!tw.next(a, t, first)) return;
        load_codes(t, false, pt, kr);
        load_groups(t, does_v, key_of, groups, g);
        const uint32_t tk = s.base + s.l.scale_k, tv = s.base + s.l.scale_v, v_bytes = kKeys * groups * 4;
        bool have_prev = false;
        for (int i = 0;; ++i) {
            if (first && have_prev) {
                emit(prev, true, vr, tv + ((i - 1) & 1) * v_bytes);
                have_prev = false;
            }
            // key factors of this tile: K by the lower 128 threads, V by the upper ones
            const int depth = i % kScaleDepth;
            wait(s, &s.sc_empty[depth], ((i / kScaleDepth) & 1) ^ 1);
            named_bar_sync(3, 32 * kProducerWarps);  // every thread is done with the tables that are rewritten
            const float top = largest(g, groups);
            if (does_v) {
                const int e = min(max(exponent(top), -15), 24);
                store_groups(tv + (i & 1) * v_bytes + key_of * groups * 4, g, groups, exp2i(kTop - e));
                reinterpret_cast<float*>(__cvta_shared_to_generic(s.base + s.l.key_v))[depth * kKeys + key_of] = e;
                const __half w = __float2half_rn(exp2i(-e));
                reinterpret_cast<__half*>(__cvta_shared_to_generic(s.base + s.l.key_w))[depth * kKeys + key_of] = w;
            } else {
                const int e = min(max(exponent(top), -100), 120);
                store_groups(tk + key_of * groups * 4, g, groups, exp2i(kTop - e));
                reinterpret_cast<float*>(__cvta_shared_to_generic(s.base + s.l.key_k))[depth * kKeys + key_of] = exp2i(e - kTop);
            }
            named_bar_sync(3, 32 * kProducerWarps);
            if (pt == 0) mbar_arrive(&s.sc_full[depth]);
            more = tw.next(a, next, next_first);
            if (more) load_groups(next, does_v, key_of, groups, g);
            emit(t, false, kr, tk);
            if (more) load_codes(next, false, pt, kr);
            if (have_prev) emit(prev, true, vr, tv + ((i - 1) & 1) * v_bytes);
            load_codes(t, true, pt, vr);
            prev = t;
            have_prev = true;
            if (!more) {
                emit(prev, true, vr, tv + (i & 1) * v_bytes);
                return;
            }
            t = next;
            first = next_first;
        }
    }

    // ------------------------------------------------------------ products
    __device__ static void issue(const Args& a, const Shared& s, Walker w, uint32_t tmem) {
        Ring ring{0, 0};
        int tile = 0, units = 0;
        Unit u;
        const uint32_t q = s.base + s.l.q, p = s.base + s.l.p;
        while (w.next(a, u)) {
            const uint32_t n = u.rows <= 64 ? 64 : kRows;
            const uint32_t desc_qk = tc5::shape(!kQuant, false, n), desc_pv = tc5::shape(!kQuant, true, n);
            wait(s, s.q_full, units & 1);
            tc5::fence_after();
            ++units;
            const auto scores = [&](int i) {
                const uint32_t d = tmem + ((tile + i) & 1) * a.nr;
                for (int b = 0; b < NB; ++b) {
                    wait(s, &s.full[ring.slot], ring.phase);
                    tc5::fence_after();
                    const uint32_t k = s.base + ring.slot * kBox, qb = q + b * a.nr * 128;
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        tc5::mma(d, tc5::operand(k + ks * 32, 16, 1024), tc5::operand(qb + ks * 32, 16, 1024), desc_qk,
                                 b + ks > 0);
                    tc5::commit(&s.empty[ring.slot]);
                    ring.step(a.slots);
                }
                tc5::commit(&s.s_full[(tile + i) & 1]);
            };
            scores(0);
            for (int i = 0; i < u.n; ++i) {
                if (i + 1 < u.n) scores(i + 1);
                wait(s, s.p_full, (tile + i) & 1);
                tc5::fence_after();
                for (int mb = 0; mb < MB; ++mb) {
                    const int slot = ring.slot;
                    int slot2 = slot;
                    wait(s, &s.full[slot], ring.phase);
                    ring.step(a.slots);
                    if (D > 64) {
                        slot2 = ring.slot;
                        wait(s, &s.full[slot2], ring.phase);
                        ring.step(a.slots);
                    }
                    tc5::fence_after();
                    const uint32_t v = s.base + slot * kBox;
#pragma unroll
                    for (int ks = 0; ks < kKeys / 16; ++ks)
                        tc5::mma(tmem + (2 + mb) * a.nr, tc5::operand(v + ks * 2048, kBox, 1024),
                                 tc5::operand(p + ks * 2048, kBox, 1024), desc_pv, i + ks > 0);
                    tc5::commit(&s.empty[slot]);
                    if (D > 64) tc5::commit(&s.empty[slot2]);
                }
                tc5::commit(s.pv_done);
            }
            tile += u.n;
        }
    }

    // ------------------------------------------------------------ softmax
    // Q of a unit: rows of the block as K-major swizzled boxes; over quantised caches as fp16 scaled by a
    // power of two per row, in the order that the unpack leaves.
    __device__ static __forceinline__ void load_q(const Args& a, const Shared& s, const Unit& u) {
        constexpr int kPieces = D / 8;
        const int tid = threadIdx.x;
        for (int idx = tid; idx < u.rows * kPieces; idx += 32 * kSoftmaxWarps) {
            const int n = idx / kPieces, c = idx % kPieces;  // a row's pieces sit in one warp
            const int r = u.block * kRows + n;
            const int64_t row = u.prefix ? r / a.G : (int64_t)u.seq * a.tokens + r / a.G;
            const uint4 x = *reinterpret_cast<const uint4*>(a.q + row * a.ld_q + (size_t)(u.head * a.G + r % a.G) * D + c * 8);
            uint4 y = x;
            if constexpr (kQuant) {
                float f[8];
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
                float m = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    f[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
                    m = fmaxf(m, fabsf(f[i]));
                }
                const uint32_t mask = __activemask();
#pragma unroll
                for (int o = 1; o < kPieces && o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(mask, m, o));
                const int e = min(max(exponent(m), -100), 120);
                const float sc = exp2i(kTop - e);
                uint32_t* p = &y.x;
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = pack2<false>(f[order<BITS>(2 * i)] * sc, f[order<BITS>(2 * i + 1)] * sc);
                if (c == 0) s.qs[n] = a.scale * 1.4426950408889634f * exp2i(e - kTop);
            }
            sts128(s.base + s.l.q + (c >> 3) * a.nr * 128 + n * 128 + (((c & 7) ^ (n & 7)) << 4), y);
        }
        if (tid < kRows) {
            const int n = tid, r = u.block * kRows + n;
            const bool live = n < u.rows;
            s.thr[n] = live ? -INFINITY : INFINITY;  // a row that is not there never raises its maximum
            s.mm[n] = -kLift;
            s.m[n] = -INFINITY;
            if (!kQuant) s.qs[n] = a.scale * 1.4426950408889634f;
            int info = 0;
            if (live && !u.prefix) {
                const int t = r / a.G;
                info = a.parents ? static_cast<int>(tree_walk(a.parents + (size_t)u.seq * a.tokens, t).path) : t;
            }
            s.rowinfo[n] = info;
        }
    }

    __device__ static void softmax(const Args& a, const Shared& s, Walker w, uint32_t tmem, int cta) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quarter = warp & 3, half = warp >> 2;
        const int key = quarter * 32 + lane, tid = threadIdx.x & 127;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const int columns = a.nr / 2, c0 = half * columns;  // this warp's columns of S^T
        const int l_cols = a.nr / 8, l0 = warp * l_cols;    // columns whose sums it forms (inside its half)
        const uint32_t ones = kQuant ? 0x3c003c00u : 0x3f803f80u;
        int tile = 0, units = 0;
        Unit u;
        while (w.next(a, u)) {
            load_q(a, s, u);
            fence_proxy_async_shared();
            tc5::fence_before();
            named_bar_sync(4, 32 * kSoftmaxWarps);
            if (threadIdx.x == 0) mbar_arrive(s.q_full);
            float lsum[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
            for (int i = 0; i < u.n; ++i, ++tile) {
                const int depth = tile % kScaleDepth;
                float ks = 1.f, ev = 0.f;
                wait(s, &s.s_full[tile & 1], (tile >> 1) & 1);
                tc5::fence_after();
                if (kQuant) {
                    wait(s, &s.sc_full[depth], (tile / kScaleDepth) & 1);
                    ks = reinterpret_cast<const float*>(__cvta_shared_to_generic(s.base + s.l.key_k))[depth * kKeys + key];
                    ev = reinterpret_cast<const float*>(__cvta_shared_to_generic(s.base + s.l.key_v))[depth * kKeys + key];
                }
                const int at = (u.t0 + i) * kKeys, k_at = at + key;
                const bool masked = at + kKeys > (u.prefix ? u.keys : u.len);
                float y[2][32];
                bool raise = false;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int n0 = c0 + 32 * c;
                    if (32 * c < columns && n0 < u.rows) {
                        tc5::ld32(tmem + lanes + (tile & 1) * a.nr + n0, y[c]);
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 th = *reinterpret_cast<const float4*>(&s.thr[n0 + j]);
                            const float4 qs = *reinterpret_cast<const float4*>(&s.qs[n0 + j]);
                            const float t4[4] = {th.x, th.y, th.z, th.w}, q4[4] = {qs.x, qs.y, qs.z, qs.w};
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                float v = kQuant ? fmaf(y[c][j + x] * ks, q4[x], ev) : y[c][j + x] * q4[x];
                                if (masked) {
                                    const int b = k_at - u.len;  // block row of the key
                                    const int info = s.rowinfo[n0 + j + x];
                                    const bool seen = k_at < u.len || (!u.prefix && k_at < u.keys &&
                                                                       (a.parents ? (info >> b) & 1 : b <= info));
                                    v = seen ? v : -INFINITY;
                                }
                                raise = raise || v > t4[x];
                                y[c][j + x] = v;
                            }
                        }
                    }
                }
                bool waited = i == 0;
                if (bar_any(1 + half, 128, raise)) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int n0 = c0 + 32 * c;
                        if (32 * c < columns && n0 < u.rows) {
                            float mine = -INFINITY;
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                const float m = warp_max(y[c][j]);
                                if (lane == j) mine = m;
                            }
                            s.part[quarter * kRows + n0 + lane] = mine;
                        }
                    }
                    named_bar_sync(1 + half, 128);
                    if (tid < columns && c0 + tid < u.rows) {
                        const int n = c0 + tid;
                        const float old = s.m[n];
                        const float m = fmaxf(fmaxf(fmaxf(s.part[n], s.part[kRows + n]),
                                                    fmaxf(s.part[2 * kRows + n], s.part[3 * kRows + n])), old);
                        s.corr[n] = m == old ? 1.f : ex2(old - m);
                        s.m[n] = m;
                        s.thr[n] = m + kLazy;
                        s.mm[n] = (m == -INFINITY ? 0.f : m) - kLift;
                    }
                    named_bar_sync(1 + half, 128);
                    if (!waited) {  // the accumulators so far go to the new maxima
                        wait(s, s.pv_done, (tile - 1) & 1);
                        tc5::fence_after();
                        waited = true;
                        if (D > 64 || quarter < 2) {
                            for (int mb = 0; mb < MB; ++mb)
                                for (int n0 = c0; n0 < min(c0 + columns, u.rows); n0 += 16) {
                                    uint32_t r[16];
                                    const uint32_t addr = tmem + lanes + (2 + mb) * a.nr + n0;
                                    tc5::ld16(addr, r);
#pragma unroll
                                    for (int j = 0; j < 16; ++j)
                                        r[j] = __float_as_uint(__uint_as_float(r[j]) * (n0 + j < u.rows ? s.corr[n0 + j] : 1.f));
                                    tc5::st16(addr, r);
                                }
                            tc5::wait_st();
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        if (8 * x < l_cols) {
                            const int n = l0 + 8 * x + 2 * (lane & 3);
                            if (n < u.rows) lsum[x][0] *= s.corr[n];
                            if (n + 1 < u.rows) lsum[x][1] *= s.corr[n + 1];
                        }
                }
                if (!waited) {
                    wait(s, s.pv_done, (tile - 1) & 1);  // P is free again
                    tc5::fence_after();
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int n0 = c0 + 32 * c;
                    if (32 * c < columns && n0 < u.rows) {
                        const uint32_t row = s.base + s.l.p + (n0 >> 6) * kBox + key * 128;
#pragma unroll
                        for (int j = 0; j < 32; j += 8) {
                            const float4 ma = *reinterpret_cast<const float4*>(&s.mm[n0 + j]);
                            const float4 mb = *reinterpret_cast<const float4*>(&s.mm[n0 + j + 4]);
                            uint4 v;
                            v.x = pack2<!kQuant>(ex2(y[c][j] - ma.x), ex2(y[c][j + 1] - ma.y));
                            v.y = pack2<!kQuant>(ex2(y[c][j + 2] - ma.z), ex2(y[c][j + 3] - ma.w));
                            v.z = pack2<!kQuant>(ex2(y[c][j + 4] - mb.x), ex2(y[c][j + 5] - mb.y));
                            v.w = pack2<!kQuant>(ex2(y[c][j + 6] - mb.z), ex2(y[c][j + 7] - mb.w));
                            sts128(row + (((((n0 & 63) + j) >> 3) ^ (key & 7)) << 4), v);
                        }
                    }
                }
                fence_proxy_async_shared();
                tc5::fence_before();
                named_bar_sync(1 + half, 128);
                if (tid == 0) mbar_arrive(s.p_full);
                // sums of the columns over the tile's keys: one 16-row product with a row of ones (or of
                // the keys' weights), on the rounded P that the numerator uses
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int n = l0 + 8 * x;
                    if (8 * x < l_cols && n < u.rows) {
                        const uint32_t box = s.base + s.l.p + (n >> 6) * kBox;
#pragma unroll
                        for (int kk = 0; kk < kKeys; kk += 32) {
                            const int r = kk + lane;
                            uint32_t b0, b1, b2, b3;
                            asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                                         : "=r"(b0), "=r"(b1), "=r"(b2), "=r"(b3)
                                         : "r"(box + r * 128 + (((((n & 63) >> 3)) ^ (r & 7)) << 4))
                                         : "memory");
                            if constexpr (kQuant) {
                                const uint32_t kw = s.base + s.l.key_w + (depth * kKeys + kk + 2 * (lane & 3)) * 2;
                                const uint32_t a0 = lds32(kw), a2 = lds32(kw + 16), a4 = lds32(kw + 32), a6 = lds32(kw + 48);
                                mma_f16_16816(lsum[x], a0, a0, a2, a2, b0, b1);
                                mma_f16_16816(lsum[x], a4, a4, a6, a6, b2, b3);
                            } else {
                                mma_bf16_16816(lsum[x], ones, ones, ones, ones, b0, b1);
                                mma_bf16_16816(lsum[x], ones, ones, ones, ones, b2, b3);
                            }
                        }
                    }
                }
                if (kQuant) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s.sc_empty[depth]);
                }
            }
            // the unit's partial
            wait(s, s.pv_done, (tile - 1) & 1);
            tc5::fence_after();
            const long long at = partial_row(a, u.prefix, u.segment, cta);
            if (D > 64 || quarter < 2) {
                for (int mb = 0; mb < MB; ++mb) {
                    const int e = mb * 128 + quarter * 32 + lane;
                    float* o = a.o + at * D + ((e & ~7) | order<BITS>(e & 7));
                    for (int n0 = c0; n0 < min(c0 + columns, u.rows); n0 += 16) {
                        uint32_t r[16];
                        tc5::ld16(tmem + lanes + (2 + mb) * a.nr + n0, r);
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (n0 + j < u.rows) o[(long long)(n0 + j) * D] = __uint_as_float(r[j]);
                    }
                }
            }
            if (lane < 4) {
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    if (8 * x < l_cols) {
                        const int n = l0 + 8 * x + 2 * lane;
                        if (n < u.rows) a.ml[at + n] = make_float2(s.m[n], lsum[x][0]);
                        if (n + 1 < u.rows) a.ml[at + n + 1] = make_float2(s.m[n + 1], lsum[x][1]);
                    }
            }
            if (threadIdx.x == 0) {
                const long long seg = (u.prefix ? 0 : segments_p(a)) + u.segment;
                if (u.t0 == 0) a.first[seg] = cta;
                if (u.t0 + u.n == u.tiles) a.last[seg] = cta;
                int* flag = &s.poison[units & (kPoison - 1)];
                a.poison[partial_index(a, u.prefix, u.segment, cta)] = *reinterpret_cast<volatile int*>(flag);
                *flag = 0;
            }
            ++units;
            tc5::fence_before();
            named_bar_sync(4, 32 * kSoftmaxWarps);  // Q, the row arrays and the accumulators are free
        }
    }

    // The CTA's run of tiles: a scan over the entries' tile counts.
    __device__ static void plan(const Args& a, int* misc) {
        const int entries = a.cache.sequences * a.blocks_o, tid = threadIdx.x;
        const int per = (entries + kThreads - 1) / kThreads;
        const int e0 = min(entries, tid * per), e1 = min(entries, e0 + per);
        const int tiles_p = (a.prefix_len + kKeys - 1) / kKeys, prefix_end = tiles_p * a.blocks_p * a.cache.hkv;
        int sum = 0;
        for (int e = e0; e < e1; ++e) {
            if (e % a.blocks_o == 0 && blockIdx.x == 0) kv::block_start(a.lengths, e / a.blocks_o, a.tokens, a.cache.max_len);
            sum += entry_tiles(a, e) * a.cache.hkv;
        }
        int* s_warp = misc + 8;
        const int warp = tid >> 5, lane = tid & 31;
        int scan = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += v;
        }
        if (lane == 31) s_warp[warp] = scan;
        __syncthreads();
        int before = prefix_end + scan - sum, total = prefix_end;
        for (int i = 0; i < kThreads / 32; ++i) {
            if (i < warp) before += s_warp[i];
            total += s_warp[i];
        }
        // with nothing but absent sequences the prefix has no reader
        if (total == prefix_end) total = 0;
        const int ctas = min(static_cast<int>(gridDim.x), total), cta = blockIdx.x;
        const int w0 = cta < ctas ? static_cast<int>((long long)total * cta / ctas) : 0;
        const int w1 = cta < ctas ? static_cast<int>((long long)total * (cta + 1) / ctas) : 0;
        const int w = max(w0, prefix_end);  // first own tile of the run
        if (tid == 0) {
            misc[2] = w0;
            misc[3] = w1;
            misc[4] = misc[5] = 0;
        }
        __syncthreads();
        if (w < w1 && before <= w && w < before + sum) {
            int off = before, e = e0, n = entry_tiles(a, e) * a.cache.hkv;
            while (w >= off + n) {
                off += n;
                n = entry_tiles(a, ++e) * a.cache.hkv;
            }
            misc[4] = e;
            misc[5] = off;
        }
    }

    __device__ static void run(const Args& a) {
        extern __shared__ __align__(1024) uint8_t smem[];
        Shared s;
        s.base = (smem_u32(smem) + 1023u) & ~1023u;
        s.l = layout(D, a.nr, a.slots, kQuant ? D / a.cache.group : 0);
        uint8_t* g = smem + (s.base - smem_u32(smem));
        s.full = reinterpret_cast<uint64_t*>(g + s.l.bars);
        s.empty = s.full + kMaxSlots;
        s.s_full = s.empty + kMaxSlots;
        s.p_full = s.s_full + 2;
        s.pv_done = s.p_full + 1;
        s.q_full = s.pv_done + 1;
        s.sc_full = s.q_full + 1;
        s.sc_empty = s.sc_full + kScaleDepth;
        s.poison = reinterpret_cast<int*>(g + s.l.misc);
        s.misc = s.poison + kPoison;
        s.abort = s.misc;
        s.thr = reinterpret_cast<float*>(g + s.l.row);
        s.mm = s.thr + kRows;
        s.qs = s.mm + kRows;
        s.corr = s.qs + kRows;
        s.m = s.corr + kRows;
        s.rowinfo = reinterpret_cast<int*>(s.m + kRows);
        s.part = reinterpret_cast<float*>(g + s.l.part);
        const int warp = threadIdx.x >> 5;
        if (threadIdx.x == 0) {
            for (int i = 0; i < kMaxSlots; ++i) {
                mbar_init(&s.full[i], kProducerWarps);
                mbar_init(&s.empty[i], 1);
            }
            mbar_init(&s.s_full[0], 1);
            mbar_init(&s.s_full[1], 1);
            mbar_init(s.p_full, 2);
            mbar_init(s.pv_done, 1);
            mbar_init(s.q_full, 1);
            for (int i = 0; i < kScaleDepth; ++i) {
                mbar_init(&s.sc_full[i], 1);
                mbar_init(&s.sc_empty[i], kSoftmaxWarps);
            }
            s.misc[0] = 0;
            fence_barrier_init();
        }
        if (threadIdx.x < kPoison) s.poison[threadIdx.x] = 0;
        if (warp == kSoftmaxWarps + kProducerWarps) tc5::alloc(smem_u32(&s.misc[1]), kTmemColumns);
        pdl_wait();
        pdl_launch_dependents();
        plan(a, s.misc);
        tc5::fence_before();
        __syncthreads();
        tc5::fence_after();
        const uint32_t tmem = *reinterpret_cast<volatile int*>(&s.misc[1]);
        const Walker w{s.misc[2], s.misc[3], s.misc[4], s.misc[5]};
        if (warp < kSoftmaxWarps) {
            softmax(a, s, w, tmem, blockIdx.x);
        } else if (warp < kSoftmaxWarps + kProducerWarps) {
            if constexpr (kQuant) produce_quant(a, s, w);
            else produce_bf16(a, s, w);
        } else {
            if ((threadIdx.x & 31) == 0) issue(a, s, w, tmem);
            __syncwarp();
        }
        tc5::fence_before();
        __syncthreads();
        if (warp == kSoftmaxWarps + kProducerWarps) tc5::dealloc(tmem, kTmemColumns);
    }
};

template <int BITS, int D>
__global__ void __launch_bounds__(kThreads, 1) attn_batch_kernel(const __grid_constant__ Args a) {
    Kernel<BITS, D>::run(a);
}

__device__ __forceinline__ float element(const kv::View& c, int64_t row, int e) {  // of V
    if (c.bits == 16) return bf16_bits_to_float(reinterpret_cast<const uint16_t*>(c.v)[row * c.d + e]);
    const int64_t g = row * (c.d / c.group) + e / c.group;
    const int code = c.bits == 8 ? c.v[row * c.d + e] : (c.v[(row * c.d + e) / 2] >> (4 * (e & 1))) & 15;
    return fmaf(bf16_bits_to_float(c.vs[g]), static_cast<float>(code), bf16_bits_to_float(c.vb[g]));
}

// Joins the partials of a row and applies the gate: one warp per (row, q head).
template <int BITS, int D>
__global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ Args a) {
    constexpr int CH = D / 32;
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= (long long)a.cache.sequences * a.tokens * a.hq) return;
    const int r = static_cast<int>(item / a.hq), h = static_cast<int>(item - (long long)r * a.hq);
    const int seq = r / a.tokens, t = r - seq * a.tokens, head = h / a.G, g = h - head * a.G;
    const int len = live_length(a, seq);
    if (len < 0) return;
    float m = -INFINITY, l = 0.f, acc[CH];
    int poison = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i) acc[i] = 0.f;
    for (int side = 0; side < 2; ++side) {
        const bool prefix = side == 0;
        if (prefix && a.blocks_p == 0) continue;
        const long long row = prefix ? (long long)r * a.G + g : (long long)t * a.G + g;
        const int block = static_cast<int>(row / kRows), n = static_cast<int>(row % kRows);
        const long long seg = prefix ? (long long)block * a.cache.hkv + head
                                     : ((long long)seq * a.blocks_o + block) * a.cache.hkv + head;
        const long long meta = (prefix ? 0 : segments_p(a)) + seg;
        const int c0 = a.first[meta], c1 = a.last[meta];
        for (int base = c0; base <= c1; base += 32) {
            const int mine = base + lane;
            float2 ml = make_float2(-INFINITY, 0.f);
            if (mine <= c1) {
                ml = a.ml[partial_row(a, prefix, seg, mine) + n];
                if (!prefix) poison |= a.poison[partial_index(a, prefix, seg, mine)];
            }
            float mx = ml.x;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float m_new = fmaxf(m, mx);
            const float old = m == m_new ? 1.f : ex2(m - m_new);
            const float w = ml.x == -INFINITY ? 0.f : ex2(ml.x - m_new);
            m = m_new;
            l *= old;
            l = fmaf(w, ml.y, l);  // summed over the lanes below
#pragma unroll
            for (int i = 0; i < CH; ++i) acc[i] *= old;
            const int count = min(32, c1 - base + 1);
            for (int j0 = 0; j0 < count; j0 += 4) {
                float x[4][CH];
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (j0 + u < count) {
                        const float* src = a.o + (partial_row(a, prefix, seg, base + j0 + u) + n) * D + lane * CH;
#pragma unroll
                        for (int i = 0; i < CH; i += 2) {
                            const float2 v = *reinterpret_cast<const float2*>(src + i);
                            x[u][i] = v.x;
                            x[u][i + 1] = v.y;
                        }
                    }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float wu = __shfl_sync(0xffffffffu, w, (j0 + u) & 31);
                    if (j0 + u < count) {
#pragma unroll
                        for (int i = 0; i < CH; ++i) acc[i] = fmaf(wu, x[u][i], acc[i]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    poison = __any_sync(0xffffffffu, poison != 0);
    const float inv = (BITS == 16 ? 1.f : exp2i(-kTop)) / l;
#pragma unroll
    for (int i = 0; i < CH; ++i) acc[i] *= inv;
    if (poison) {  // block rows whose values were taken out: they reach the rows that see them
        const uint32_t path = a.parents ? tree_walk(a.parents + (size_t)seq * a.tokens, t).path : 0u;
        for (int b = 0; b < a.tokens; ++b) {
            if (a.parents ? !((path >> b) & 1u) : b > t) continue;
            const int64_t row = kv::row_index(a.cache, seq, head, len + b);
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const float v = element(a.cache, row, lane * CH + i);
                if (!(fabsf(v) < INFINITY)) acc[i] += v;
            }
        }
    }
    uint16_t* out = a.out + (size_t)r * a.hq * D + (size_t)h * D + lane * CH;
    if (a.gate) {
        float gt[CH];
        kv::load_lane<CH>(a.gate + (size_t)r * a.ld_gate + (size_t)h * D + lane * CH, gt);
#pragma unroll
        for (int i = 0; i < CH; ++i) acc[i] /= 1.f + __expf(-gt[i]);
    }
    kv::store_lane<CH>(out, acc);
}

static int check(const dflash_kv_cache* cache, const dflash_kv_cache* prefix, int prefix_len, int tokens, int hq,
                 const char* who) {
    const int st = kv::check_cache(cache, who);
    if (st != DFLASH_OK) return st;
    if (tokens < 1 || tokens > cache->max_len || hq < 1 || hq % cache->kv_heads || prefix_len < 0)
        return fail(DFLASH_ERR_INVALID_ARGUMENT, "%s: bad arguments", who);
    const long long G = hq / cache->kv_heads, tiles = (cache->max_len + kKeys - 1ll) / kKeys;
    const long long blocks_p = prefix_len ? ((long long)cache->sequences * tokens * G + kRows - 1) / kRows : 0;
    const long long blocks_o = ((long long)tokens * G + kRows - 1) / kRows;
    if (G > 64 || (long long)cache->sequences * tokens > 0x7fffffffll / hq ||
        (long long)prefix_len + cache->max_len > 0x7fffffffll - kKeys ||
        blocks_p * cache->kv_heads * ((prefix_len + kKeys - 1ll) / kKeys) +
                cache->sequences * blocks_o * cache->kv_heads * tiles > 0x7fffffffll)
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

// Sizes of a checked call and, with a base, its workspace pointers; returns the workspace's bytes.
static size_t fit(Args& a, const dflash_kv_cache& c, int prefix_len, int tokens, int hq, uint8_t* base) {
    a.cache = kv::view_of(c);
    a.prefix_len = prefix_len;
    a.tokens = tokens;
    a.hq = hq;
    a.G = hq / c.kv_heads;
    const long long rows_p = (long long)c.sequences * tokens * a.G, rows_o = (long long)tokens * a.G;
    a.blocks_p = prefix_len ? static_cast<int>((rows_p + kRows - 1) / kRows) : 0;
    a.blocks_o = static_cast<int>((rows_o + kRows - 1) / kRows);
    a.rows_o = static_cast<int>(rows_o < kRows ? rows_o : kRows);
    a.nr = (prefix_len ? rows_p : rows_o) <= 64 ? 64 : kRows;
    const int groups = c.bits == 16 ? 0 : c.head_dim / c.group;
    a.slots = kMaxSlots;
    while (layout(c.head_dim, a.nr, a.slots, groups).total > kSmemLimit) a.slots -= 2;
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        uint8_t* p = base + at;
        at += (bytes + 15) / 16 * 16;
        return p;
    };
    const size_t segs = segments_p(a) + segments_o(a), parts = partials_p(a) + partials_o(a);
    const size_t rows = partials_p(a) * kRows + partials_o(a) * a.rows_o;
    a.first = reinterpret_cast<int32_t*>(take(4 * segs));
    a.last = reinterpret_cast<int32_t*>(take(4 * segs));
    a.poison = reinterpret_cast<int32_t*>(take(4 * parts));
    a.ml = reinterpret_cast<float2*>(take(8 * rows));
    a.o = reinterpret_cast<float*>(take(4 * rows * c.head_dim));
    return at;
}

template <int BITS, int D>
static cudaError_t launch(const Args& a, int ctas, cudaStream_t s) {
    const int groups = BITS == 16 ? 0 : D / a.cache.group;
    const size_t smem = layout(D, a.nr, a.slots, groups).total + 1024;
    cudaError_t e = cudaFuncSetAttribute(attn_batch_kernel<BITS, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
    if (e != cudaSuccess) return e;
    e = launch_chained(attn_batch_kernel<BITS, D>, dim3(ctas), dim3(kThreads), smem, s, 1, a);
    if (e != cudaSuccess) return e;
    const long long items = (long long)a.cache.sequences * a.tokens * a.hq;
    return launch_chained(attn_join_kernel<BITS, D>, dim3(static_cast<unsigned>((items + 7) / 8)), dim3(256), 0, s, 1, a);
}

}  // namespace attn
}  // namespace dflash

extern "C" size_t dflash_stack_attn_decode_batch_workspace_bytes(const dflash_kv_cache* cache, int prefix_len, int tokens,
                                                                 int hq) {
    using namespace dflash;
    if (attn::check(cache, nullptr, prefix_len, tokens, hq, "dflash_stack_attn_decode_batch_workspace_bytes") != DFLASH_OK)
        return 0;
    attn::Args a{};
    return attn::fit(a, *cache, prefix_len, tokens, hq, nullptr);
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
    const int d = cache->head_dim;
    if (!q || !lengths || !out || (parents && tokens > kMaxTreeRows) || (prefix_len > 0 && !prefix) ||
        ld_q < (long long)hq * d || (gate && ld_gate < (long long)hq * d))
        return fail(DFLASH_ERR_INVALID_ARGUMENT, "%s: bad arguments", who);
    if (!kv::stride_ok(q, ld_q, 1) || (gate && !kv::stride_ok(gate, ld_gate, 1)) || !aligned16(out))
        return fail(DFLASH_ERR_MISALIGNED, "%s: q, gate, out and their row strides must be 16-byte aligned", who);
    attn::Args a{};
    const size_t need = attn::fit(a, *cache, prefix_len, tokens, hq, static_cast<uint8_t*>(workspace));
    if (!workspace || workspace_bytes < need || !aligned16(workspace))
        return fail(DFLASH_ERR_WORKSPACE, "%s: needs %zu bytes of 16-byte aligned workspace", who, need);
    a.q = q;
    a.gate = gate;
    a.out = out;
    a.ld_q = ld_q;
    a.ld_gate = ld_gate;
    a.prefix = kv::view_of(prefix_len > 0 ? *prefix : *cache);
    a.lengths = lengths;
    a.parents = parents;
    a.scale = scale;
    int dev = 0;
    DFLASH_CUDA_TRY(cudaGetDevice(&dev));
    // no more CTAs than tiles that the lengths can give
    const long long most = attn::segments_p(a) * ((prefix_len + attn::kKeys - 1) / attn::kKeys) +
                           attn::segments_o(a) * ((cache->max_len + attn::kKeys - 1ll) / attn::kKeys);
    long long ctas = sm_count(dev) < attn::kMaxCtas ? sm_count(dev) : attn::kMaxCtas;
    if (ctas > most) ctas = most;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e = cudaErrorInvalidValue;
#define DFLASH_BATCH_CASE(BITS, D) \
    if (cache->bits == BITS && d == D) e = attn::launch<BITS, D>(a, static_cast<int>(ctas), s);
    DFLASH_BATCH_CASE(16, 64) DFLASH_BATCH_CASE(16, 128) DFLASH_BATCH_CASE(16, 256)
    DFLASH_BATCH_CASE(8, 64) DFLASH_BATCH_CASE(8, 128) DFLASH_BATCH_CASE(8, 256)
    DFLASH_BATCH_CASE(4, 64) DFLASH_BATCH_CASE(4, 128) DFLASH_BATCH_CASE(4, 256)
#undef DFLASH_BATCH_CASE
    DFLASH_CUDA_TRY(e);
    return DFLASH_OK;
}
