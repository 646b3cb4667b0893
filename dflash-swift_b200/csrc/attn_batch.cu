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
// one key: its mask and its scale factors are its own registers.
//
// Q, K, V and P are bf16 over bf16 caches: a product takes one type for both operands, and the cache's range is not fp16's.
// P's rounding to 2^-9 is the price (0.0023 of the output against 64 bits, where the output's own rounding is 0.0017 and
// dflash_stack_attn_decode's fp32 weights add nothing).  P in two parts would cost half as much product again and 32 KB of
// shared memory, one of three ring slots at 256 dims; a sum of the rounded P gained nothing (0.0023) and took 2 % more time.
// Over quantised caches they are fp16, whose 11 bits lose little to the codes' 8: every
// key's values (and every query row) are first scaled by a power of two into fp16's upper range,
// undone in S^T for K and Q, and for V folded into P's exponent and the sum's weights.
//
// Roles: first the softmax warps (per TMEM lane quarter two or four, 32 columns each), then the producers (cache
// rows to swizzled shared memory boxes of 128 keys x 64 elements, in rings; over quantised caches half of
// them for K and half for V), warp 24 issues the products, warps 25 and 26 the bulk copies of K's and V's
// codes to staging slots (27 has no work).  The running maximum is only raised when a score passes it by
// kLazy (in powers of two), so the accumulators are rarely rescaled.
//
// Measured in a captured graph, join included (256 dims, 24 q heads on 4 kv heads, groups of 64): a block of 8 tokens
// over 1024 rows of 8 bits 18.4 us; over 131071 rows 107 us (2.7 TB/s; HBM alone would take 44); 33 sequences of one token
// over about 4096 rows of 4 bits 93 us; 64 sequences of 4 tokens that share 32768 bf16 rows 245 us (0.84 PFLOP/s) in a
// short run, 265 to 280 us once the GPU has been under such load for a second (graph and call alike); with
// 128 dims, 16 q heads on 2 kv heads, 2 x 509 tokens over about 7000 rows of 8 bits 149 us.  Over quantised caches no
// unit is full (131071 rows: instructions, mostly the unpack's and the softmax's, take 56 % of the issue slots, shared memory's
// banks are 29 % busy, the tensor cores 16 %): the chain from codes to boxes to S to P to O, which two or three slots
// overlap only in part, bounds it.  Over bf16 caches the products take about half of a tile's time, the rest is the same
// chain and the change of units.  Both have some 25 us beside their tiles: launch, first loads, the changes of units
// (5 us each) and the join (11 us there).
#include "common.cuh"
#include "dflash_batch.h"
#include "tcgen05.cuh"

#include <atomic>
#include <cstddef>

namespace dflash {
namespace attn {

constexpr int kKeys = 128;
constexpr int kRows = 128;
constexpr int kBox = kKeys * 128;          // bytes of a box: 128 keys x 64 elements of 16 bits
constexpr int kIssueWarp = 24;             // behind the softmax and producer warps, 8 of one and 16 of the other
constexpr int kThreads = 32 * (kIssueWarp + 4);  // whole warpgroups: registers move between them
// Registers a thread at launch, and behind setmaxnreg for the issuing warpgroup; the producers give too, and what the
// softmax takes is no more than that, so nobody waits for good.
constexpr int kLaunchRegs = 72, kIssueRegs = 40;
constexpr int kMaxCtas = 160;              // partials are sized for this many CTAs
constexpr int kMaxSlots = 10;              // ring slots: two boxes each, one where d is 64
constexpr int kMaxStages = 8;              // staging slots for codes: 64 or 128 rows each
constexpr int kScaleDepth = 2;             // tiles whose key factors may be alive at once
// Tiles that the change to another unit of a sequence counts as in the plan.  Counting none leaves SMs with many short units
// far behind; beyond that the number was picked from two shapes, is not monotone (it moves the runs' borders), and weighs a
// tile of few rows like one of 128 and a change within the prefix as nothing.  64 sequences of 200 rows behind a bf16 prefix of
// 32768: 451 us with none, 287 with 1, 295 with 2, 254 with 4, 308 with 6; 32 of 250 rows behind 8190 of 8 bits: 47.3, 40.5,
// 41.0, 47.5 with none, 1, 2 and 4 (long sequences: 92.7, 93.2, 92.1, 91.4).
__host__ __device__ constexpr int unit_cost(int bits) { return bits == 16 ? 4 : 2; }
constexpr int kPoison = 16;                // units whose poison flags may be alive at once
constexpr float kLazy = 4.f;               // a maximum moves when a score passes it by 2^4 ...
constexpr float kNever = 3e38f;            // base of a row without a maximum yet: every score passes it
// A key's factor 2^e goes into its P and out of its sum's weight, so P of two keys may be 2^(e - e') apart at the same score:
// exact sums as long as the values' sizes differ by no more than 2^126, which ex2 and the join's weights reach.
constexpr int kZero = -62;                 // exponent of a row of zeros: halfway, so beside sizes of 2^-84 to 2^64
constexpr float kTiny = 2.350988701644575e-38f;  // 2^-125: smaller rows (top is a quarter) count as zeros
constexpr int kTopQ = 12;                  // query rows are scaled to 2^12 .. 2^13 in fp16
constexpr uint32_t kTmemColumns = 512;
constexpr int kAllSoftmax = 5;               // named barrier of all softmax warps; 1 to 4: of those with the same columns
constexpr int kSmemLimit = 232448;

// Shared memory: what has a fixed size first, so that its addresses are constants; then the scale
// tables, and from the next 1024-byte border on the ring, Q and P.
struct Fixed {
    uint64_t full[kMaxSlots], empty[kMaxSlots], s_full[2], p_full, pv_done, q_full, sc_full[kScaleDepth],
        sc_empty[kScaleDepth], staged[kMaxStages], unstaged[kMaxStages], drained;
    alignas(16) float base[kRows];      // -(maximum - kLift): scores are taken relative to it; read four at a time, like qs
    float qs[kRows], corr[kRows], m[kRows];
    int info[kRows];                    // chain: the row's token; tree: its path mask
    float part[4][kRows];
    float key_k[kScaleDepth][kKeys], key_v[kScaleDepth][kKeys];
    int poison[kPoison];
    int abort, tmem, w0, w1, entry, off, pad;
    int unit_tiles, unit_rows;          // for the issuing thread, from the softmax warps
    int warp_sum[2][kThreads / 32];
};
static_assert(offsetof(Fixed, base) % 16 == 0 && offsetof(Fixed, qs) % 16 == 0 &&
                  alignof(Fixed) == 16, "vector accesses");
constexpr uint32_t kTables = (sizeof(Fixed) + 15) / 16 * 16;

struct Layout {
    uint32_t ring, q, p, stage, total;
};
__host__ inline Layout layout(int d, int nr, int slots, int stages, int stage_bytes, int groups) {
    Layout l;
    l.ring = (kTables + 3 * kKeys * groups * 4 + 1023) / 1024 * 1024;
    l.q = l.ring + slots * (d > 64 ? 2 : 1) * kBox;
    l.p = l.q + nr * d * 2;
    l.stage = l.p + kKeys * nr * 2;
    l.total = l.stage + stages * stage_bytes;
    return l;
}

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
    int G, g_magic;              // q heads per kv head, and 2^16 / G rounded up
    int blocks_p, blocks_o;      // row blocks of the prefix and of one sequence
    int rows_o;                  // rows of a block of one sequence, at most
    int rb;                      // query rows of a block: kRows or 64
    int nr;                      // columns of the products' buffers: 64 or kRows
    int slots_k, slots;          // ring slots: K's and all of them (quantised caches; one ring over bf16 caches)
    int stages, stage_rows;      // staging slots of K, as many of V, and their rows (quantised caches)
    Layout l;
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
    return prefix ? (segment + cta) * a.rb : partials_p(a) * a.rb + (segment + cta) * a.rows_o;
}
__device__ __forceinline__ long long partial_index(const Args& a, bool prefix, long long segment, int cta) {
    return prefix ? segment + cta : partials_p(a) + segment + cta;
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
    if (a.parents || block + 1 == a.blocks_o) return len + a.tokens;
    return len + ((block + 1) * a.rb - 1) / a.G + 1;
}
__device__ __forceinline__ int live_length(const Args& a, int seq) {
    const int n = a.lengths[seq];
    return n > a.cache.max_len - a.tokens ? -1 : n;
}
__device__ __forceinline__ int entry_tiles(const Args& a, int e) {
    const int seq = a.blocks_o == 1 ? e : e / a.blocks_o, len = live_length(a, seq);  // most often one block: no division
    return len < 0 ? 0 : (own_keys(a, len, e - seq * a.blocks_o) + kKeys - 1) / kKeys;
}

// A run counts places: a tile of the prefix is one, and a (row block, kv head) of a sequence has `pad` of them before its
// tiles', so that a run with many short units has fewer tiles.
struct Walker {
    int w, w1;          // next place and end of the run
    int entry, off;     // own region: current (sequence, row block) and its first place
    int pad;
    __device__ __forceinline__ bool next(const Args& a, Unit& u) {
        if (w >= w1) return false;
        const int tiles_p = (a.prefix_len + kKeys - 1) / kKeys, prefix_end = tiles_p * a.blocks_p * a.cache.hkv;
        if (w < prefix_end) {
            const int s = w / tiles_p;
            u.prefix = true;
            u.segment = s;
            u.block = s / a.cache.hkv;
            u.head = s - u.block * a.cache.hkv;
            u.seq = 0;
            u.tiles = tiles_p;
            u.t0 = w - s * tiles_p;
            u.rows = min(a.rb, a.cache.sequences * a.tokens * a.G - u.block * a.rb);
            u.len = u.keys = a.prefix_len;
            u.n = min(tiles_p - u.t0, w1 - w);
            w += u.n;
        } else {
            int tiles = entry_tiles(a, entry), places = tiles ? tiles + pad : 0;
            while (w >= off + places * a.cache.hkv) {
                off += places * a.cache.hkv;
                tiles = entry_tiles(a, ++entry);
                places = tiles ? tiles + pad : 0;
            }
            const int rel = w - off;
            u.prefix = false;
            u.head = rel / places;
            u.seq = a.blocks_o == 1 ? entry : entry / a.blocks_o;
            u.block = entry - u.seq * a.blocks_o;
            u.segment = (long long)entry * a.cache.hkv + u.head;
            u.tiles = tiles;
            const int first = rel - u.head * places - pad;  // below 0: places without a tile
            u.t0 = max(first, 0);
            u.rows = min(a.rb, a.tokens * a.G - u.block * a.rb);
            u.len = a.lengths[u.seq];
            u.keys = own_keys(a, u.len, u.block);
            const int left = min(tiles - first, w1 - w);  // places of the run in here
            w += left;
            u.n = left + min(first, 0);
            if (u.n <= 0) return false;  // the run ends before the first tile
        }
        return true;
    }
};

// ---------------------------------------------------------------- small helpers
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two 32-bit operations in one instruction: a *= b, a += b, a = a * b + c.
__device__ __forceinline__ void mul2(float& a0, float& a1, float b0, float b1) {
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
        "mul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}" : "+f"(a0), "+f"(a1) : "f"(b0), "f"(b1));
}
__device__ __forceinline__ void add2(float& a0, float& a1, float b0, float b1) {
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
        "add.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}" : "+f"(a0), "+f"(a1) : "f"(b0), "f"(b1));
}
__device__ __forceinline__ void fma2(float& a0, float& a1, float b0, float b1, float c0, float c1) {
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tmov.b64 c, {%4, %5};\n\t"
        "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "+f"(a0), "+f"(a1) : "f"(b0), "f"(b1), "f"(c0), "f"(c1));
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
__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool fill) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(fill ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// Arrives on the mbarrier (one of its expected arrivals) once this thread's copies so far are complete.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Copies `bytes` (a multiple of 16, 16-byte aligned on both sides) to shared memory; they count on the mbarrier.
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
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
__device__ __forceinline__ float exp2_any(int e) {  // 2^e, e in -149 .. 127
    return e < -126 ? __int_as_float(1 << (e + 149)) : exp2i(e);
}
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
    // Keys are scaled to 2^kTop .. 2^(kTop + 1): the step of a group, at most 2^(kTop + 2) / (2^BITS - 1), has
    // to stay under 2^-8 (store_groups).  An element under 2^(-14 - kTop) of its key's largest is subnormal in fp16 and
    // held to 2^(-25 - kTop) of that.
    static constexpr int kTop = BITS == 8 ? -3 : -7;
    // P is 2^kLift p, and up to 2^kLazy more: in fp16 2^8, so that small weights stay normal; in bf16, which has fp32's range,
    // 2^-16, so that the sum of p V over 2^12 keys stays in range for values up to the largest.
    static constexpr float kLift = kQuant ? 8.f : -16.f;
    // 16 softmax warps, four per TMEM lane quarter with 32 columns each, and 8 producers; over quantised caches of 256
    // dims, whose row blocks have 64 rows (all their columns belong to eight warps) and whose codes take twice the
    // unpacking, 8 and 16.  (1018 tokens over 7000 rows of 8 bits and 128 dims: 150 us with sixteen, 175 with eight.)
    static constexpr int kSoftmaxWarps = kQuant && D == 256 ? 8 : 16, kSubs = kSoftmaxWarps / 4;
    static constexpr int kProducerWarps = kIssueWarp - kSoftmaxWarps;
    static constexpr int kGroupWarps = kQuant ? kProducerWarps / 2 : kProducerWarps, kGroup = 32 * kGroupWarps;  // that fill a box
    static constexpr int kProducerRegs = kQuant ? kSoftmaxWarps == 8 ? 64 : 72 : 48;
    static constexpr int kSoftmaxRegs =
        (32 * (28 * kLaunchRegs - 4 * kIssueRegs - kProducerWarps * kProducerRegs) / (32 * kSoftmaxWarps)) / 8 * 8;
    static constexpr int NB = D / 64;                  // boxes of a K or V tile
    static constexpr int MB = D > 64 ? D / 128 : 1;    // 128-lane blocks of O^T (half used when d is 64) = ring slots of a tile
    static constexpr int kSub = NB / MB, kSlot = kSub * kBox;  // boxes and bytes of a ring slot

    __device__ static __forceinline__ Fixed& fixed() {
        extern __shared__ __align__(1024) uint8_t smem[];
        return *reinterpret_cast<Fixed*>(smem);
    }
    __device__ static __forceinline__ uint32_t smem_at(uint32_t offset) { return smem_u32(&fixed()) + offset; }

    // A bounded wait that stays small where it is inlined: a failed try sleeps for as long as the hardware
    // lets it (the phase's end wakes it), and 2^22 of them raise the error.  No clock is read, whose read
    // costs more than the usual wait.  After an error every wait returns at once and the roles run on to
    // their ends; copies and products in flight are drained there, since the block's shared and tensor memory
    // must not go, to another block perhaps, before them (0.2 us a call: the drains themselves find nothing to wait for).
    __device__ static __forceinline__ bool aborted() { return *const_cast<volatile int*>(&fixed().abort) != 0; }
    __device__ static __forceinline__ void give_up() {
        atomicOr(&g_device_error, DFLASH_DEVERR_ATTN_PIPELINE);
        *const_cast<volatile int*>(&fixed().abort) = 1;
    }
    __device__ static __forceinline__ void wait(uint64_t* bar, uint32_t parity) {
        if (mbar_try_wait(bar, parity)) return;
        for (int n = 0; !mbar_try_wait(bar, parity); ++n) {
            if (aborted()) return;
            if (n == 1 << 22) give_up();
        }
    }
    __device__ static __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
        for (int n = 0; n < 1 << 22 && !mbar_try_wait(bar, parity); ++n) {
        }
    }

    // ------------------------------------------------------------ producers
    // The products take K(0), then K(i) V(i - 1), then V(n - 1) of a unit.
    struct Ring {
        int slot, first, end;
        uint32_t phase;
        __device__ __forceinline__ void step() {
            if (++slot == end) {
                slot = first;
                phase ^= 1;
            }
        }
    };
    // K's and V's ring: one ring for both over bf16 caches, whose producers fill it in the products' order; one each
    // where two groups of producers fill them, since a wait by parity only tells a phase from the one before it
    // and a group must not run ahead of the other's use of a slot.
    __device__ static __forceinline__ Ring ring_of(const Args& a, bool is_v) {
        return kQuant && is_v ? Ring{a.slots_k, a.slots_k, a.slots, 0} : Ring{0, 0, a.slots_k, 0};
    }

    // Where the rows of a unit's (sequence, kv head) lie.
    struct Source {
        const uint8_t *k, *v;
        int64_t row0;
        bool prefix;
        int keys;    // rows that exist and that some query row sees
        int hidden;  // rows from here on are hidden from some query row
        int t0, n;
        __device__ __forceinline__ Source() {}
        __device__ __forceinline__ Source(const Args& a, const Unit& u) {
            const kv::View& c = u.prefix ? a.prefix : a.cache;
            row0 = kv::row_index(c, u.seq, u.head, 0);
            k = c.k + row0 * (D * BITS / 8);
            v = c.v + row0 * (D * BITS / 8);
            prefix = u.prefix;
            keys = u.keys;
            hidden = u.prefix ? u.keys : u.len;
            t0 = u.t0;
            n = u.n;
        }
    };

    // The writes become visible to the tensor cores through the proxy fence of the thread that waits for
    // them (issue): a fence here would wait for this warp's loads in flight as well.
    __device__ static __forceinline__ void signal_full(int slot) {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&fixed().full[slot]);
    }

    // The pieces of a box that a producer thread writes: kPieces rows, kChunks 16-byte chunks of each.
    static constexpr int kChunks = kQuant ? 16 / BITS : 1;
    static constexpr int kRowThreads = kQuant ? BITS / 2 : 8;  // threads that share a row
    static constexpr int kRowStep = kGroup / kRowThreads, kPieces = kKeys / kRowStep;
    __device__ static __forceinline__ int piece_key(int pt, int u) { return pt / kRowThreads + u * kRowStep; }

    // A non-finite element of a row that some query row does not see would reach it as 0 * inf: it is
    // taken out of the operand and the unit's flag raised, for the join to put it back where it is
    // seen.  Each thread looks at what it wrote itself.
    __device__ static __forceinline__ void take_out(uint32_t box, int from, int pt, int* flag) {
        constexpr uint32_t kExp = kQuant ? 0x7c00u : 0x7f80u;
#pragma unroll 1
        for (int u = 0; u < kPieces * kChunks; ++u) {
            const int key = piece_key(pt, u / kChunks), chunk = (pt % kRowThreads) * kChunks + u % kChunks;
            if (key < from) continue;
            const uint32_t addr = box + key * 128 + ((chunk ^ (key & 7)) << 4);
            const uint4 x = lds128(addr);
            uint32_t w[4] = {x.x, x.y, x.z, x.w};
            bool bad = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if ((w[i] & kExp) == kExp) { w[i] &= 0xffff0000u; bad = true; }
                if ((w[i] & (kExp << 16)) == (kExp << 16)) { w[i] &= 0x0000ffffu; bad = true; }
            }
            if (bad) {
                sts128(addr, make_uint4(w[0], w[1], w[2], w[3]));
                *reinterpret_cast<volatile int*>(flag) = 1;
            }
        }
    }

    // bf16 caches: cp.async straight into the swizzled boxes; the copies themselves arrive on the box's
    // barrier, so as many boxes are in flight as the ring has free slots.
    __device__ static void produce_bf16(const Args& a, Walker w) {
        const int pt = threadIdx.x - 32 * kSoftmaxWarps, key0 = pt >> 3, c = pt & 7;
        const uint32_t ring_at = smem_at(a.l.ring), dst0 = ring_at + key0 * 128 + ((c ^ (key0 & 7)) << 4);
        Ring ring = ring_of(a, false);
        Unit u;
        for (int unit = 0; w.next(a, u); ++unit) {
            const Source src(a, u);
#pragma unroll 1
            for (int step = 1; step <= 2 * src.n; ++step) {  // K0 K1 V0 K2 V1 .. V(n-1)
                const bool is_v = step > 1 && (step == 2 * src.n || (step & 1));
                const int i = is_v ? (step == 2 * src.n ? src.n - 1 : step / 2 - 1) : step / 2;
                const int key_at = (src.t0 + i) * kKeys, valid = min(kKeys, src.keys - key_at);
                const int look = max(0, src.hidden - key_at);
                const uint8_t* p = (is_v ? src.v : src.k) + ((int64_t)(key_at + key0) * D + c * 8) * 2;
#pragma unroll 1
                for (int b = 0; b < MB; ++b, p += kSub * 128) {
                    wait(&fixed().empty[ring.slot], ring.phase ^ 1);
#pragma unroll
                    for (int x = 0; x < kPieces; ++x) {
                        const bool live = key0 + kRowStep * x < valid;
#pragma unroll
                        for (int y = 0; y < kSub; ++y)
                            cp_async16(dst0 + ring.slot * kSlot + y * kBox + x * kRowStep * 128,
                                       live ? p + x * (kRowStep * D * 2) + y * 128 : src.k, live);
                    }
                    if (__builtin_expect(is_v && look < valid, 0)) {
                        cp_async_wait_all();
                        for (int y = 0; y < kSub; ++y)
                            take_out(ring_at + ring.slot * kSlot + y * kBox, look, pt, &fixed().poison[unit & (kPoison - 1)]);
                        mbar_arrive(&fixed().full[ring.slot]);
                    } else {
                        cp_async_arrive(&fixed().full[ring.slot]);
                    }
                    ring.step();
                }
            }
        }
        cp_async_wait_all();  // nothing is in flight when the block's shared memory goes
    }

    // Quantised caches: a lane each for K and V copies runs of rows to their staging slots with bulk copies, a
    // group of producers each unpacks the codes to fp16 boxes.  Rows behind the last one stay whatever
    // the slot held: their scale and bias are 0.
    __device__ static void stage(const Args& a, Walker w, bool is_v) {
        const uint32_t slot_bytes = a.stage_rows * (D * BITS / 8);
        const int first = is_v ? a.stages : 0;
        Unit u;
        int slot = first;
        uint32_t phase = 0;
        while (w.next(a, u)) {
            const Source src(a, u);
            const uint8_t* rows = is_v ? src.v : src.k;
#pragma unroll 1
            for (int at = src.t0 * kKeys; at < (src.t0 + src.n) * kKeys; at += a.stage_rows) {
                // as wait(), but no copy goes to a slot that was not handed back
                bool mine = mbar_try_wait(&fixed().unstaged[slot], phase ^ 1);
#pragma unroll 1
                for (int n = 0; !mine; ++n) {
                    if (aborted()) goto out;
                    if (n == 1 << 22) give_up();
                    mine = mbar_try_wait(&fixed().unstaged[slot], phase ^ 1);
                }
                const uint32_t bytes = min(a.stage_rows, max(0, src.keys - at)) * (D * BITS / 8);
                mbar_arrive_expect_tx(&fixed().staged[slot], bytes);
                if (bytes)
                    bulk_copy(smem_at(a.l.stage) + slot * slot_bytes, rows + (int64_t)at * (D * BITS / 8), bytes,
                              &fixed().staged[slot]);
                if (++slot == first + a.stages) {
                    slot = first;
                    phase ^= 1;
                }
            }
        }
out:
#pragma unroll 1
        for (int i = first; i < first + a.stages; ++i) drain(&fixed().staged[i], i < slot ? phase : phase ^ 1);
    }

    // Scales and biases of one key, as raw bf16 pairs: up to two words of each, of four where a key has
    // eight groups (256 dims) and two lanes, for one lane.
    struct Groups {
        uint32_t s[2], b[2];
    };
    __device__ static __forceinline__ void load_groups(const Args& a, const Source& src, bool is_v, int key, int groups,
                                                       int first, Groups& g) {
        const kv::View& c = src.prefix ? a.prefix : a.cache;
        const int64_t at = (src.row0 + key) * groups;
        const uint16_t *ps = (is_v ? c.vs : c.ks) + at, *pb = (is_v ? c.vb : c.kb) + at;
#pragma unroll
        for (int i = 0; i < 2; ++i) g.s[i] = g.b[i] = 0;
        if (key >= src.keys) return;
        if (groups == 1) {
            if (first == 0) {
                g.s[0] = *ps;
                g.b[0] = *pb;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (2 * (first + i) < groups && (i == 0 || groups == 8 || kGroupWarps == 4)) {
                    g.s[i] = reinterpret_cast<const uint32_t*>(ps)[first + i];
                    g.b[i] = reinterpret_cast<const uint32_t*>(pb)[first + i];
                }
        }
    }
    // A quarter of the largest magnitude that a lane's groups can stand for (the whole could pass fp32's range by a rounding).
    __device__ static __forceinline__ float largest(const Groups& g) {
        constexpr float kCodes = BITS == 8 ? 63.75f : 3.75f;
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // zero where there is none
            const float s0 = __uint_as_float(g.s[i] << 16), s1 = __uint_as_float(g.s[i] & 0xffff0000u);
            const float b0 = 0.25f * __uint_as_float(g.b[i] << 16), b1 = 0.25f * __uint_as_float(g.b[i] & 0xffff0000u);
            m = largest_of(m, b0, fmaf(kCodes, s0, b0));
            m = largest_of(m, b1, fmaf(kCodes, s1, b1));
        }
        return m;
    }
    __device__ static __forceinline__ float largest_of(float m, float x, float y) {  // NaN stays NaN
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(m), "f"(fabsf(x)));
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(m), "f"(fabsf(y)));
        return m;
    }
    // Table entries (fp16 scale * f * 2^24, bias * f): a code in the low bits of a half is the subnormal
    // code * 2^-24, so that one fma gives scale * code + bias (|scale * f| < 2^-8: see kTop).
    __device__ static __forceinline__ void store_groups(uint32_t addr, const Groups& g, int groups, int first, float f) {
        const float f24 = f * 16777216.f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (2 * (first + i) < groups && (i == 0 || groups == 8 || kGroupWarps == 4)) {
                const uint32_t e0 = pack2<false>(__uint_as_float(g.s[i] << 16) * f24, __uint_as_float(g.b[i] << 16) * f);
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr + 8 * (first + i)), "r"(e0) : "memory");
                if (groups > 1) {
                    const uint32_t e1 = pack2<false>(__uint_as_float(g.s[i] & 0xffff0000u) * f24,
                                                     __uint_as_float(g.b[i] & 0xffff0000u) * f);
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr + 8 * (first + i) + 4), "r"(e1) : "memory");
                }
            }
    }
    // Unpacks one 16-byte piece (32 or 16 elements of one key and group) to its chunks of a box row.
    __device__ static __forceinline__ void unpack(uint4 codes, uint32_t sb, uint32_t row, const uint32_t (&chunk)[kChunks]) {
        const uint32_t s2 = __byte_perm(sb, 0, 0x1010), b2 = __byte_perm(sb, 0, 0x3232);
        const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
        if constexpr (BITS == 4) {
            const uint32_t t2 = mul_h2(s2, 0x2c002c00u);  // 2^-4: codes four bits further up
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t hi = w[i] >> 8;
                sts128(row + chunk[i], make_uint4(fma_h2(w[i] & 0x000f000fu, s2, b2), fma_h2(w[i] & 0x00f000f0u, t2, b2),
                                                  fma_h2(hi & 0x000f000fu, s2, b2), fma_h2(hi & 0x00f000f0u, t2, b2)));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                sts128(row + chunk[i], make_uint4(fma_h2(__byte_perm(w[2 * i], 0, 0x4140), s2, b2),
                                                  fma_h2(__byte_perm(w[2 * i], 0, 0x4342), s2, b2),
                                                  fma_h2(__byte_perm(w[2 * i + 1], 0, 0x4140), s2, b2),
                                                  fma_h2(__byte_perm(w[2 * i + 1], 0, 0x4342), s2, b2)));
        }
    }

    __device__ static void produce_quant(const Args& a, Walker w, bool is_v) {
        const int pt = threadIdx.x & (kGroup - 1), groups = D / a.cache.group;
        const int piece = pt % kRowThreads, key0 = pt / kRowThreads;
        const uint32_t ring_at = smem_at(a.l.ring), slot_bytes = a.stage_rows * (D * BITS / 8);
        const int shift = 31 - __clz(a.cache.group);
        // A quarter-warp reads the same columns of two (8 bits) or four (4 bits) rows, which would lie in the same
        // banks: every other row takes the two boxes of a slot in the other order.
        constexpr int kRowBytes = D * BITS / 8;
        const int mix = kSub == 1 ? 0 : (kRowBytes >= 128 ? key0 : key0 >> 1) & 1;
        uint32_t chunk[kChunks];
#pragma unroll
        for (int i = 0; i < kChunks; ++i) chunk[i] = key0 * 128 + (((kChunks * piece + i) ^ (key0 & 7)) << 4);
        const uint32_t from = smem_at(a.l.stage) + key0 * kRowBytes + piece * 16;
        const bool halves = a.stage_rows < kKeys;
        // Scales: a warp unpacks the same keys of every tile, so it keeps their tables for itself, one or two lanes a key.
        // V's are made a tile ahead of its unpacking, since the softmax needs V's factor.
        constexpr int kOwn = kKeys / kGroupWarps, kRun = 32 / kRowThreads;  // keys of a warp, in runs of kRun
        const int lane = threadIdx.x & 31, kk = lane % kOwn, first = groups == 8 ? 2 * (lane / kOwn) : lane / kOwn;
        const int key_of = (pt >> 5) * kRun + kk % kRun + kk / kRun * kRowStep;
        const uint32_t table_bytes = kKeys * groups * 4, tables = smem_at(kTables) + (is_v ? table_bytes : 0);
        Groups g;
        Ring ring = ring_of(a, is_v);
        const int first_slot = is_v ? a.stages : 0;
        int slot = first_slot;
        uint32_t phase = 0;
        // look: first row of the tile to look at for non-finite values, kKeys for none
        const auto emit = [&](uint32_t table, int look, int unit) {
            uint32_t codes[2];  // the tile's rows 0 and 64 on: one slot, or two halves
            int staged[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if (x == 0 || halves) {
                    staged[x] = slot;
                    codes[x] = from + slot * slot_bytes;
                    wait(&fixed().staged[slot], phase);
                    if (++slot == first_slot + a.stages) {
                        slot = first_slot;
                        phase ^= 1;
                    }
                } else {
                    codes[x] = codes[0] + kKeys / 2 * kRowBytes;
                }
            }
            const uint32_t entry = table + key0 * groups * 4;
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                wait(&fixed().empty[ring.slot], ring.phase ^ 1);
                const uint32_t box0 = ring_at + ring.slot * kSlot;
#pragma unroll
                for (int b = 0; b < kSub; ++b) {
                    const int mine = b ^ mix, box = m * kSub + mine;  // the box this thread's row takes now
                    const uint32_t sb = entry + ((box * 64 + piece * (128 / BITS)) >> shift) * 4;
#pragma unroll
                    for (int x = 0; x < kPieces; ++x)
                        unpack(lds128(codes[x * kRowStep / 64] + x * kRowStep % 64 * kRowBytes + box * (8 * BITS)), lds32(sb + x * kRowStep * groups * 4),
                               box0 + mine * kBox + x * kRowStep * 128, chunk);
                }
                if (__builtin_expect(look < kKeys, 0))
#pragma unroll 1
                    for (int b = 0; b < kSub; ++b) take_out(box0 + b * kBox, look, pt, &fixed().poison[unit & (kPoison - 1)]);
                signal_full(ring.slot);
                ring.step();
            }
            if ((threadIdx.x & 31) == 0) {  // the codes have been read
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    if (x == 0 || halves) mbar_arrive(&fixed().unstaged[staged[x]]);
            }
        };
        Unit u;
        if (!w.next(a, u)) return;
        Source cur(a, u), next;
        load_groups(a, cur, is_v, cur.t0 * kKeys + key_of, groups, first, g);
        int tile = 0;
        bool more = true, bad = false;
        for (int unit = 0; more; ++unit) {
            more = w.next(a, u);
            if (more) next = Source(a, u);
#pragma unroll 1
            for (int i = 0; i <= cur.n; ++i, ++tile) {  // K(i), V(i - 1)
                const bool bad_before = bad;
                if (i < cur.n) {
                    const int depth = tile % kScaleDepth;
                    wait(&fixed().sc_empty[depth], ((tile / kScaleDepth) & 1) ^ 1);
                    float top = largest(g);
                    if constexpr (kOwn == 16) {
                        const float other = __shfl_xor_sync(0xffffffffu, top, 16);
                        asm("max.NaN.f32 %0, %1, %2;" : "=f"(top) : "f"(top), "f"(other));
                    }
                    // Every finite size up to the largest: 2^(kTop - e) may be subnormal, which a product takes as it is.
                    // A row of zeros, whose exponent could be any, counts as smaller than what it lies beside (V's goes
                    // into the maxima, and must not hold those of small rows up), but no smaller than kZero: its
                    // weight is the softmax's still.
                    const int e = !(top < INFINITY) ? 0 : top < kTiny ? kZero : min(max(exponent(top) + 2, -100), 127);
                    store_groups(tables + (is_v ? (tile & 1) * table_bytes : 0) + key_of * groups * 4, g, groups, first,
                                 exp2_any(kTop - e));
                    if (lane < kOwn) {
                        if (is_v) {
                            fixed().key_v[depth][key_of] = e;
                        } else {
                            fixed().key_k[depth][key_of] = exp2i(e - kTop - kTopQ);
                        }
                    }
                    bad = __any_sync(0xffffffffu, !(top < INFINITY));
                    __syncwarp();  // the lanes' tables and factors, for the others and through lane 0's arrival (a vote orders nothing)
                    if (lane == 0) mbar_arrive(&fixed().sc_full[depth]);
                    if (i + 1 < cur.n) load_groups(a, cur, is_v, (cur.t0 + i + 1) * kKeys + key_of, groups, first, g);
                    else if (more) load_groups(a, next, is_v, next.t0 * kKeys + key_of, groups, first, g);
                    if (!is_v) emit(tables, kKeys, 0);
                }
                if (is_v && i > 0) {
                    const int at = (cur.t0 + i - 1) * kKeys, look = max(0, cur.hidden - at);
                    emit(tables + ((tile - 1) & 1) * table_bytes, bad_before && at + look < cur.keys ? look : kKeys, unit);
                }
            }
            --tile;  // the unit's last pass was V alone
            cur = next;
        }
    }

    // ------------------------------------------------------------ products
    // Run by a whole warp, so that addresses and descriptors stay in uniform registers; one elected lane
    // issues.  What comes from shared memory is broadcast for the same reason.
    __device__ static void issue(const Args& a, uint32_t tmem_lane) {
        const bool one = tc5::elect();
        const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_lane, 0);
        Ring rk = ring_of(a, false), rv_own = ring_of(a, true);
        Ring& rv = kQuant ? rv_own : rk;
        int tile = 0;
        const uint32_t q = smem_at(a.l.q), p = smem_at(a.l.p);
#pragma unroll 1
        for (int unit = 0;; ++unit) {
            wait(&fixed().q_full, unit & 1);
            tc5::fence_after();
            const int tiles = __shfl_sync(0xffffffffu, *const_cast<volatile int*>(&fixed().unit_tiles), 0);
            const int rows = __shfl_sync(0xffffffffu, *const_cast<volatile int*>(&fixed().unit_rows), 0);
            const uint32_t n = rows <= 64 ? 64 : kRows;
            if (tiles == 0) return;
            const uint32_t desc_qk = tc5::shape(!kQuant, false, n), desc_pv = tc5::shape(!kQuant, true, n);
            const auto scores = [&](int i) {
                const uint32_t d = tmem + ((tile + i) & 1) * a.nr;
#pragma unroll 1
                for (int b = 0; b < MB; ++b) {
                    wait(&fixed().full[rk.slot], rk.phase);
                    fence_proxy_async_shared();
                    const uint32_t k = smem_at(a.l.ring) + rk.slot * kSlot, qb = q + b * kSub * a.nr * 128;
                    const uint64_t dk = tc5::operand(k, 16, 1024), dq = tc5::operand(qb, 16, 1024);
                    const uint32_t q_step = a.nr * 128 / 16;
                    if (one) {
#pragma unroll
                        for (int y = 0; y < kSub; ++y)
#pragma unroll
                            for (int ks = 0; ks < 4; ++ks)  // 32 bytes on
                                tc5::mma(d, dk + y * (kBox / 16) + ks * 2, dq + y * q_step + ks * 2, desc_qk, b + y + ks > 0);
                        tc5::commit(&fixed().empty[rk.slot]);
                    }
                    rk.step();
                }
                if (one) tc5::commit(&fixed().s_full[(tile + i) & 1]);
            };
#pragma unroll 1
            for (int i = -1; i < tiles; ++i) {
                if (i + 1 < tiles) scores(i + 1);
                if (i < 0) continue;
                wait(&fixed().p_full, (tile + i) & 1);
                tc5::fence_after();
#pragma unroll 1
                for (int mb = 0; mb < MB; ++mb) {
                    const int slot = rv.slot;
                    wait(&fixed().full[slot], rv.phase);
                    rv.step();
                    fence_proxy_async_shared();
                    const uint64_t dv = tc5::operand(smem_at(a.l.ring) + slot * kSlot, kBox, 1024);
                    const uint64_t dp = tc5::operand(p, kBox, 1024);
                    const uint32_t d = tmem + (2 + mb) * a.nr;
                    if (one) {
#pragma unroll
                        for (int ks = 0; ks < kKeys / 16; ++ks)  // 16 keys of 128 bytes on
                            tc5::mma(d, dv + ks * 128, dp + ks * 128, desc_pv, i + ks > 0);
                        tc5::commit(&fixed().empty[slot]);
                    }
                }
                if (one) tc5::commit(&fixed().pv_done);
            }
            tile += tiles;
        }
    }

    // ------------------------------------------------------------ softmax
    // Q of a unit: rows of the block as K-major swizzled boxes; over quantised caches as fp16 scaled by a
    // power of two per row, in the order that the unpack leaves.
    __device__ static __forceinline__ void load_q(const Args& a, const Unit& u) {
        constexpr int kPer = D / 8, kBatch = 4;  // 16-byte pieces of a row, which sit in one warp; loads in flight
        const int tid = threadIdx.x;
        const int t0 = u.block ? u.block * a.rb / a.G : 0, g0 = u.block * a.rb - t0 * a.G;
        const uint16_t* base = a.q + ((u.prefix ? 0 : (int64_t)u.seq * a.tokens) + t0) * a.ld_q + (size_t)u.head * a.G * D;
        // row n of the block is token t0 + v / G, head v % G of v = g0 + n < 256: a product with 2^16 / G
        const auto token_of = [&](int n) { return static_cast<int>(static_cast<uint32_t>((g0 + n) * a.g_magic) >> 16); };
        for (int first = 0; first < u.rows * kPer; first += 32 * kSoftmaxWarps * kBatch) {
            uint4 x[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int idx = first + k * 32 * kSoftmaxWarps + tid, n = idx / kPer, c = idx % kPer;
                x[k] = make_uint4(0, 0, 0, 0);
                if (n < u.rows) {
                    const int t = token_of(n);
                    x[k] = *reinterpret_cast<const uint4*>(base + t * a.ld_q + (g0 + n - t * a.G) * D + c * 8);
                }
            }
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int idx = first + k * 32 * kSoftmaxWarps + tid, n = idx / kPer, c = idx % kPer;
                uint4 y = x[k];
                if constexpr (kQuant) {
                    float f[8];
                    const uint32_t w[4] = {y.x, y.y, y.z, y.w};
                    float m = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        f[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
                        m = fmaxf(m, fabsf(f[i]));
                    }
#pragma unroll
                    for (int o = 1; o < kPer; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                    const int e = max(exponent(m), kTopQ - 126);
                    const float sc = exp2i(kTopQ - e);
                    uint32_t* p = &y.x;
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[i] = pack2<false>(f[order<BITS>(2 * i)] * sc, f[order<BITS>(2 * i + 1)] * sc);
                    if (c == 0 && n < u.rows) fixed().qs[n] = a.scale * 1.4426950408889634f * exp2i(e);
                }
                if (n < u.rows) sts128(smem_at(a.l.q) + (c >> 3) * a.nr * 128 + n * 128 + (((c & 7) ^ (n & 7)) << 4), y);
            }
        }
        if (tid < kRows) {
            const int n = tid;
            const bool live = n < u.rows;
            fixed().base[n] = live ? kNever : -INFINITY;  // nothing passes that of a row that is not there
            fixed().m[n] = -INFINITY;
            // key b of the block (below 0: cached rows) is seen if b <= info, in a tree if bit b of info is set
            int info = -1;
            if (live && !u.prefix) {
                const int t = t0 + token_of(n);
                info = a.parents ? static_cast<int>(tree_walk(a.parents + (size_t)u.seq * a.tokens, t).path) : t;
            }
            fixed().info[n] = info;
        }
    }

    __device__ static void softmax(const Args& a, Walker w, uint32_t tmem, int cta) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quarter = warp & 3, sub = warp >> 2;
        const int key = quarter * 32 + lane, tid = threadIdx.x & 127;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const int n0 = sub * 32;  // this warp's 32 columns of S^T
        const float qscale = a.scale * 1.4426950408889634f;
        int tile = 0, units = 0;
        Unit u;
        while (w.next(a, u)) {
            load_q(a, u);
            fence_proxy_async_shared();
            tc5::fence_before();
            named_bar_sync(kAllSoftmax, 32 * kSoftmaxWarps);
            if (threadIdx.x == 0) {
                fixed().unit_tiles = u.n;
                fixed().unit_rows = u.rows;
                mbar_arrive(&fixed().q_full);
            }
            const bool live = n0 < u.rows;
            float sum = 0.f;  // over this warp's keys, lane j has column n0 + j
            for (int i = 0; i < u.n; ++i, ++tile) {
                const int depth = tile % kScaleDepth;
                float ks = 1.f, ev = 0.f;
                wait(&fixed().s_full[tile & 1], (tile >> 1) & 1);
                tc5::fence_after();
                if (kQuant) {
                    wait(&fixed().sc_full[depth], (tile / kScaleDepth) & 1);
                    ks = fixed().key_k[depth][key];
                    ev = fixed().key_v[depth][key];
                }
                const int at = (u.t0 + i) * kKeys;
                const int b = at + key - u.len;  // block row of the key; a prefix ends where its block would begin
                const bool masked = at + kKeys > u.len;
                const float weight = kQuant ? exp2_any(-static_cast<int>(ev)) : 1.f;
                bool waited = i == 0;  // for the last tile's p V: P and the accumulators are free
                const auto hand_over = [&]() {
                    fence_proxy_async_shared();
                    tc5::fence_before();
                    named_bar_sync(1 + sub, 128);
                    if (tid == 0) mbar_arrive(&fixed().p_full);
                };
                if (live) {
                    float y[32];
                    bool raise = false;  // this pass: plain scores for new maxima, not scores relative to the old ones
#pragma unroll 1
                    for (int pass = 0;; ++pass) {  // one, or three with a raise: scores, plain scores, scores
                        tc5::ld32(tmem + lanes + (tile & 1) * a.nr + n0, y);
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            float4 bs = *reinterpret_cast<const float4*>(&fixed().base[n0 + j]);
                            if (raise) bs = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (kQuant) {
                                float4 qs = *reinterpret_cast<const float4*>(&fixed().qs[n0 + j]);
                                add2(bs.x, bs.y, ev, ev);
                                add2(bs.z, bs.w, ev, ev);
                                mul2(qs.x, qs.y, ks, ks);  // the factors first: each with y alone could pass fp32's range
                                mul2(qs.z, qs.w, ks, ks);
                                fma2(y[j], y[j + 1], qs.x, qs.y, bs.x, bs.y);
                                fma2(y[j + 2], y[j + 3], qs.z, qs.w, bs.z, bs.w);
                            } else {
                                fma2(y[j], y[j + 1], qscale, qscale, bs.x, bs.y);
                                fma2(y[j + 2], y[j + 3], qscale, qscale, bs.z, bs.w);
                            }
                        }
                        if (masked) {  // by the row's token, or its path's bits (load_q)
                            if (a.parents && !u.prefix) {
                                const int bit = b < 0 ? -1 : b < 32 ? 1 << b : 0;
#pragma unroll
                                for (int j = 0; j < 32; ++j) y[j] = fixed().info[n0 + j] & bit ? y[j] : -INFINITY;
                            } else {
#pragma unroll
                                for (int j = 0; j < 32; ++j) y[j] = b <= fixed().info[n0 + j] ? y[j] : -INFINITY;
                            }
                        }
                        if (!raise) {
                            float top[4] = {y[0], y[1], y[2], y[3]};  // NaN counts as nothing
#pragma unroll
                            for (int j = 4; j < 32; ++j) top[j & 3] = fmaxf(top[j & 3], y[j]);
                            if (pass == 0)
                                raise = bar_any(1 + sub, 128,
                                                fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) > kLazy + kLift);
                            if (!waited) {
                                wait(&fixed().pv_done, (tile - 1) & 1);
                                tc5::fence_after();
                                waited = true;
                            }
                            if (!raise) break;
                            continue;
                        }
                        raise = false;
                        float mine = -INFINITY;
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const float m = warp_max(y[j]);
                            if (lane == j) mine = m;
                        }
                        fixed().part[quarter][n0 + lane] = mine;
                        named_bar_sync(1 + sub, 128);
                        if (tid < 32 && n0 + tid < u.rows) {
                            const int n = n0 + tid;
                            const float old = fixed().m[n];
                            const float m = fmaxf(fmaxf(fmaxf(fixed().part[0][n], fixed().part[1][n]),
                                                        fmaxf(fixed().part[2][n], fixed().part[3][n])), old);
                            fixed().corr[n] = m == old ? 1.f : ex2(old - m);
                            fixed().m[n] = m;
                            if (m > -INFINITY) fixed().base[n] = kLift - m;
                        }
                        named_bar_sync(1 + sub, 128);
                        if (i > 0 && (D > 64 || quarter < 2)) {  // the accumulators so far go to the new maxima
                            for (int mb = 0; mb < MB; ++mb)
                                for (int n1 = n0; n1 < min(n0 + 32, u.rows); n1 += 16) {
                                    uint32_t r[16];
                                    const uint32_t addr = tmem + lanes + (2 + mb) * a.nr + n1;
                                    tc5::ld16(addr, r);
#pragma unroll
                                    for (int j = 0; j < 16; ++j)
                                        r[j] = __float_as_uint(__uint_as_float(r[j]) *
                                                               (n1 + j < u.rows ? fixed().corr[n1 + j] : 1.f));
                                    tc5::st16(addr, r);
                                }
                            tc5::wait_st();
                        }
                        if (n0 + lane < u.rows) sum *= fixed().corr[n0 + lane];  // and the sums
                    }
                    const uint32_t row = smem_at(a.l.p) + (n0 >> 6) * kBox + key * 128;
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {
#pragma unroll
                        for (int x = 0; x < 8; ++x) y[j + x] = ex2(y[j + x]);
                        sts128(row + (((((n0 & 63) + j) >> 3) ^ (key & 7)) << 4),
                               make_uint4(pack2<!kQuant>(y[j], y[j + 1]), pack2<!kQuant>(y[j + 2], y[j + 3]),
                                          pack2<!kQuant>(y[j + 4], y[j + 5]), pack2<!kQuant>(y[j + 6], y[j + 7])));
                    }
                    hand_over();  // before the sums, which nobody waits for
                    if (kQuant) {  // V's factor is part of P
#pragma unroll
                        for (int j = 0; j < 32; j += 2) mul2(y[j], y[j + 1], weight, weight);
                    }
                    sum += stack::reduce_scatter32(y, lane);
                } else {
                    if (i > 0) {
                        wait(&fixed().pv_done, (tile - 1) & 1);
                        tc5::fence_after();
                    }
                    hand_over();
                }
                if (kQuant) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&fixed().sc_empty[depth]);
                }
            }
            // the unit's partial
            wait(&fixed().pv_done, (tile - 1) & 1);
            tc5::fence_after();
            const long long at = partial_row(a, u.prefix, u.segment, cta);
            if (D > 64 || quarter < 2) {
                for (int mb = 0; mb < MB; ++mb) {
                    const int e = mb * 128 + quarter * 32 + lane;
                    float* o = a.o + at * D + ((e & ~7) | order<BITS>(e & 7));
                    for (int n1 = n0; n1 < min(n0 + 32, u.rows); n1 += 16) {
                        uint32_t r[16];
                        tc5::ld16(tmem + lanes + (2 + mb) * a.nr + n1, r);
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (n1 + j < u.rows) o[(long long)(n1 + j) * D] = __uint_as_float(r[j]);
                    }
                }
            }
            if (live) fixed().part[quarter][n0 + lane] = sum;
            named_bar_sync(1 + sub, 128);
            if (tid < 32 && n0 + tid < u.rows) {
                const int n = n0 + tid;
                a.ml[at + n] = make_float2(fixed().m[n], (fixed().part[0][n] + fixed().part[1][n]) +
                                                             (fixed().part[2][n] + fixed().part[3][n]));
            }
            if (threadIdx.x == 0) {
                const long long seg = (u.prefix ? 0 : segments_p(a)) + u.segment;
                if (u.t0 == 0) a.first[seg] = cta;
                if (u.t0 + u.n == u.tiles) a.last[seg] = cta;
                int* flag = &fixed().poison[units & (kPoison - 1)];
                a.poison[partial_index(a, u.prefix, u.segment, cta)] = *reinterpret_cast<volatile int*>(flag);
                *flag = 0;
            }
            ++units;
            tc5::fence_before();
            named_bar_sync(kAllSoftmax, 32 * kSoftmaxWarps);  // Q, the row arrays and the accumulators are free
        }
        if (threadIdx.x == 0) {
            fixed().unit_tiles = 0;
            mbar_arrive(&fixed().q_full);
        }
    }

    // The CTA's run of tiles: a scan over the entries' tile counts.
    __device__ static void plan(const Args& a) {
        const int entries = a.cache.sequences * a.blocks_o, tid = threadIdx.x;
        const int per = (entries + kThreads - 1) / kThreads;
        const int e0 = min(entries, tid * per), e1 = min(entries, e0 + per);
        const int tiles_p = (a.prefix_len + kKeys - 1) / kKeys, prefix_end = tiles_p * a.blocks_p * a.cache.hkv;
        int sum = 0, live = 0;
        for (int e = e0; e < e1; ++e) {
            if (e % a.blocks_o == 0 && blockIdx.x == 0) kv::block_start(a.lengths, e / a.blocks_o, a.tokens, a.cache.max_len);
            const int tiles = entry_tiles(a, e);
            sum += tiles * a.cache.hkv;
            live += tiles ? a.cache.hkv : 0;
        }
        const int warp = tid >> 5, lane = tid & 31;
        int scan = sum, scan_live = live;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, scan, o), x = __shfl_up_sync(0xffffffffu, scan_live, o);
            if (lane >= o) {
                scan += v;
                scan_live += x;
            }
        }
        if (lane == 31) {
            fixed().warp_sum[0][warp] = scan;
            fixed().warp_sum[1][warp] = scan_live;
        }
        __syncthreads();
        int before = prefix_end + scan - sum, before_live = scan_live - live, total = prefix_end, all_live = 0;
        for (int i = 0; i < kThreads / 32; ++i) {
            if (i < warp) {
                before += fixed().warp_sum[0][i];
                before_live += fixed().warp_sum[1][i];
            }
            total += fixed().warp_sum[0][i];
            all_live += fixed().warp_sum[1][i];
        }
        // no places without tiles where each CTA has one tile at most: they would put two into some
        const int pad = total > static_cast<int>(gridDim.x) ? unit_cost(BITS) : 0;
        sum += live * pad;
        before += before_live * pad;
        // with nothing but absent sequences the prefix has no reader
        total = all_live ? total + all_live * pad : 0;
        const int ctas = min(static_cast<int>(gridDim.x), total), cta = blockIdx.x;
        const auto share = [&](int c) {  // floor(total c / ctas)
            return total < (1 << 23) ? static_cast<int>(static_cast<uint32_t>(total * c) / static_cast<uint32_t>(ctas))
                                     : static_cast<int>((long long)total * c / ctas);
        };
        const int w0 = cta < ctas ? share(cta) : 0, w1 = cta < ctas ? share(cta + 1) : 0;
        const int w = max(w0, prefix_end);  // first own tile of the run
        if (tid == 0) {
            fixed().w0 = w0;
            fixed().w1 = w1;
            fixed().entry = fixed().off = 0;
            fixed().pad = pad;
        }
        __syncthreads();
        if (w < w1 && before <= w && w < before + sum) {
            const auto places = [&](int x) {
                const int tiles = entry_tiles(a, x);
                return tiles ? (tiles + pad) * a.cache.hkv : 0;
            };
            int off = before, e = e0, n = places(e);
            while (w >= off + n) {
                off += n;
                n = places(++e);
            }
            fixed().entry = e;
            fixed().off = off;
        }
    }

    __device__ static void run(const Args& a) {
        if (smem_at(0) & 1023u) {  // the swizzled boxes need it; every thread leaves here
            if (threadIdx.x == 0) atomicOr(&g_device_error, DFLASH_DEVERR_ATTN_PIPELINE);
            return;
        }
        const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
        if (threadIdx.x == 0) {
            for (int i = 0; i < kMaxSlots; ++i) {
                mbar_init(&fixed().full[i], kQuant ? kGroupWarps : kGroup);
                mbar_init(&fixed().empty[i], 1);
            }
            mbar_init(&fixed().s_full[0], 1);
            mbar_init(&fixed().s_full[1], 1);
            mbar_init(&fixed().p_full, kSubs);
            mbar_init(&fixed().pv_done, 1);
            mbar_init(&fixed().q_full, 1);
            mbar_init(&fixed().drained, 1);
            for (int i = 0; i < kScaleDepth; ++i) {
                mbar_init(&fixed().sc_full[i], kProducerWarps);
                mbar_init(&fixed().sc_empty[i], kSoftmaxWarps);
            }
            for (int i = 0; i < kMaxStages; ++i) {
                mbar_init(&fixed().staged[i], 1);
                mbar_init(&fixed().unstaged[i], kGroupWarps);
            }
            fixed().abort = fixed().unit_tiles = 0;
            fence_barrier_init();
        }
        if (threadIdx.x < kPoison) fixed().poison[threadIdx.x] = 0;
        if (warp == kIssueWarp) tc5::alloc(smem_u32(&fixed().tmem), kTmemColumns);
        pdl_wait();
        pdl_launch_dependents();
        plan(a);
        tc5::fence_before();
        __syncthreads();
        tc5::fence_after();
        const uint32_t tmem = *reinterpret_cast<volatile int*>(&fixed().tmem);
        const Walker w{fixed().w0, fixed().w1, fixed().entry, fixed().off, fixed().pad};
        if (warp < kSoftmaxWarps) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
            softmax(a, w, tmem, blockIdx.x);
        } else if (warp < kIssueWarp) {
            if constexpr (kProducerRegs < kLaunchRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegs));
            if constexpr (kQuant) produce_quant(a, w, warp >= kSoftmaxWarps + kGroupWarps);
            else produce_bf16(a, w);
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
            if (warp == kIssueWarp) issue(a, tmem);
            else if (kQuant && (warp == kIssueWarp + 1 || warp == kIssueWarp + 2) && (threadIdx.x & 31) == 0)
                stage(a, w, warp == kIssueWarp + 2);
            __syncwarp();
        }
        tc5::fence_before();
        __syncthreads();
        if (warp == kIssueWarp) {
            if (aborted()) {  // else the softmax has waited for every product
                if (tc5::elect()) tc5::commit(&fixed().drained);
                drain(&fixed().drained, 0);
            }
            tc5::dealloc(tmem, kTmemColumns);
        }
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

// Joins the partials of a row and applies the gate.  `ways` warps of a CTA share a (row, q head): all eight
// where that leaves few CTAs idle, one where there are rows enough (the reads of a partial are one dependent
// chain of a few hundred nanoseconds each otherwise).  With the attention before it, eight against one: 192 (row, head)
// pairs over 1 k keys 17.6 us and 18.9, over 131 k keys 104 and 119; a prompt's 16288 pairs 216 and 149.
template <int BITS, int D>
__global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ Args a, int ways) {
    constexpr int CH = D / 32, kWarps = 8;
    __shared__ float s_m[kWarps], s_l[kWarps], s_acc[kWarps][D];
    __shared__ int s_poison[kWarps];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, way = ways == 1 ? 0 : warp;
    const long long item = ways == 1 ? (long long)blockIdx.x * kWarps + warp : blockIdx.x;
    if (item >= (long long)a.cache.sequences * a.tokens * a.hq) return;  // whole warps, and where ways is 8 never
    const int r = static_cast<int>(item / a.hq), h = static_cast<int>(item - (long long)r * a.hq);
    const int seq = r / a.tokens, t = r - seq * a.tokens, head = h / a.G, g = h - head * a.G;
    const int len = live_length(a, seq);
    if (len < 0) return;  // every warp of the item
    float m = -INFINITY, l = 0.f, acc[CH];
    int poison = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i) acc[i] = 0.f;
    for (int side = 0; side < 2; ++side) {
        const bool prefix = side == 0;
        if (prefix && a.blocks_p == 0) continue;
        const long long row = prefix ? (long long)r * a.G + g : (long long)t * a.G + g;
        const int block = static_cast<int>(row / a.rb), n = static_cast<int>(row - (long long)block * a.rb);
        const long long seg = prefix ? (long long)block * a.cache.hkv + head
                                     : ((long long)seq * a.blocks_o + block) * a.cache.hkv + head;
        const long long meta = (prefix ? 0 : segments_p(a)) + seg;
        const int c0 = a.first[meta] + way, c1 = a.last[meta];
        for (int base = c0; base <= c1; base += 32 * ways) {
            const int mine = base + lane * ways;
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
            const int count = min(32, (c1 - base) / ways + 1);
            for (int j0 = 0; j0 < count; j0 += 4) {
                float x[4][CH];
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (j0 + u < count) {
                        const float* src = a.o + (partial_row(a, prefix, seg, base + (j0 + u) * ways) + n) * D + lane * CH;
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
    if (ways > 1) {  // the warps' parts, in order
        if (lane == 0) {
            s_m[warp] = m;
            s_l[warp] = l;
            s_poison[warp] = poison;
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) s_acc[warp][lane * CH + i] = acc[i];
        __syncthreads();
        if (warp != 0) return;
        poison = 0;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) poison |= s_poison[k];
        float mx = s_m[0];
#pragma unroll
        for (int k = 1; k < kWarps; ++k) mx = fmaxf(mx, s_m[k]);
        l = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i) acc[i] = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
            const float w = s_m[k] == -INFINITY ? 0.f : ex2(s_m[k] - mx);
            l = fmaf(w, s_l[k], l);
#pragma unroll
            for (int i = 0; i < CH; ++i) acc[i] = fmaf(w, s_acc[k][lane * CH + i], acc[i]);
        }
    }
    const float inv = (BITS == 16 ? 1.f : exp2i(-Kernel<BITS, D>::kTop)) / l;
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

// Query rows of a block: kRows, but 64 over quantised caches of 256 dims, where Q and P of 128 rows would leave the codes no
// room in shared memory.
static int row_block(const dflash_kv_cache& c) { return c.bits != 16 && c.head_dim == 256 ? 64 : kRows; }

static int check(const dflash_kv_cache* cache, const dflash_kv_cache* prefix, int prefix_len, int tokens, int hq,
                 const char* who) {
    const int st = kv::check_cache(cache, who);
    if (st != DFLASH_OK) return st;
    if (tokens < 1 || tokens > cache->max_len || hq < 1 || hq % cache->kv_heads || prefix_len < 0)
        return fail(DFLASH_ERR_INVALID_ARGUMENT, "%s: bad arguments", who);
    const long long G = hq / cache->kv_heads, rb = row_block(*cache), tiles = (cache->max_len + kKeys - 1ll) / kKeys;
    const long long blocks_p = prefix_len ? ((long long)cache->sequences * tokens * G + rb - 1) / rb : 0;
    const long long blocks_o = ((long long)tokens * G + rb - 1) / rb;
    if (G > 64 || (long long)cache->sequences * tokens > 0x7fffffffll / hq ||
        (long long)prefix_len + cache->max_len > 0x7fffffffll - kKeys ||
        blocks_p * cache->kv_heads * ((prefix_len + kKeys - 1ll) / kKeys) +
                cache->sequences * blocks_o * cache->kv_heads * (tiles + unit_cost(cache->bits)) > 0x7fffffffll)
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
    a.g_magic = (65536 + a.G - 1) / a.G;  // v / G exactly for v < 256, G <= 64: v (G - 1) < 2^16
    a.rb = row_block(c);
    const long long rows_p = (long long)c.sequences * tokens * a.G, rows_o = (long long)tokens * a.G;
    a.blocks_p = prefix_len ? static_cast<int>((rows_p + a.rb - 1) / a.rb) : 0;
    a.blocks_o = static_cast<int>((rows_o + a.rb - 1) / a.rb);
    a.rows_o = static_cast<int>(rows_o < a.rb ? rows_o : a.rb);
    a.nr = a.rb == 64 || (prefix_len ? rows_p : rows_o) <= 64 ? 64 : kRows;
    const int groups = c.bits == 16 ? 0 : c.head_dim / c.group;
    // bf16: all that fits in ring slots.  Quantised: as many slots of two for K and two for V as leave each two
    // staging slots, of whole tiles or (8 bits) of halves: two, since one would wait out each copy's latency.
    const int sub = c.head_dim > 64 ? 2 : 1, row_bytes = c.head_dim * c.bits / 8;
    const auto fits = [&](int slots, int stages, int rows) {
        return layout(c.head_dim, a.nr, slots, stages, rows * row_bytes, groups).total <= kSmemLimit;
    };
    a.stages = 0;
    a.stage_rows = kKeys;
    if (c.bits == 16) {
        a.slots = kMaxSlots / sub;
        while (!fits(a.slots, 0, 0)) --a.slots;
        a.slots_k = a.slots;
    } else {
        for (a.slots = 4; a.slots >= 2 && a.stages == 0; --a.slots)
            for (int rows = kKeys; rows >= (c.bits == 8 ? kKeys / 2 : kKeys) && a.stages == 0; rows /= 2)
                for (int n = kMaxStages / 2; n >= 2 && a.stages == 0; --n)
                    if (fits(a.slots, 2 * n, rows)) {
                        a.stages = n;
                        a.stage_rows = rows;
                    }
        ++a.slots;
        a.slots_k = a.slots / 2;  // of three, two for V: its products wait for P, K's run a tile ahead
    }
    a.l = layout(c.head_dim, a.nr, a.slots, 2 * a.stages, a.stage_rows * row_bytes, groups);
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        uint8_t* p = base + at;
        at += (bytes + 15) / 16 * 16;
        return p;
    };
    const size_t segs = segments_p(a) + segments_o(a), parts = partials_p(a) + partials_o(a);
    const size_t rows = partials_p(a) * a.rb + partials_o(a) * a.rows_o;
    a.first = reinterpret_cast<int32_t*>(take(4 * segs));
    a.last = reinterpret_cast<int32_t*>(take(4 * segs));
    a.poison = reinterpret_cast<int32_t*>(take(4 * parts));
    a.ml = reinterpret_cast<float2*>(take(8 * rows));
    a.o = reinterpret_cast<float*>(take(4 * rows * c.head_dim));
    return at;
}

template <int BITS, int D>
static cudaError_t launch(const Args& a, int ctas, cudaStream_t s) {
    static std::atomic<unsigned long long> ready{0};  // devices that know the kernel's shared memory, a bit each
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !((ready.load() >> dev) & 1)) {
        e = cudaFuncSetAttribute(attn_batch_kernel<BITS, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(1ull << dev);
    }
    e = launch_chained(attn_batch_kernel<BITS, D>, dim3(ctas), dim3(kThreads), a.l.total, s, 1, a);
    if (e != cudaSuccess) return e;
    const long long items = (long long)a.cache.sequences * a.tokens * a.hq;
    const int ways = items <= 8ll * ctas ? 8 : 1;
    return launch_chained(attn_join_kernel<BITS, D>, dim3(static_cast<unsigned>(ways == 1 ? (items + 7) / 8 : items)), dim3(256), 0,
                          s, 1, a, ways);
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
