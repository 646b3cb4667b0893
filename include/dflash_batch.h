/*
 * libdflashcuda — batches of sequences over attention caches of 16, 8 or 4 bits, a prefix
 * that the sequences share, and the log probabilities of tokens.
 *
 * The entries of dflash_stack.h run one sequence over a bf16 cache; these run `sequences`
 * of them, each with `tokens` block rows (row b * tokens + t is token t of sequence b).
 * Conventions as there: device pointers, one row per token, stream-ordered, status return,
 * capturable in a CUDA graph; the current device is the one that owns the tensors.  The
 * reference holds one sequence and a bf16 cache (the target's caches of
 * Sources/DFlashKit/DFlashSpeculativeGenerator.swift:389-398) and has no counterpart.
 */
#ifndef DFLASH_BATCH_H
#define DFLASH_BATCH_H

#include "dflash_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The attention caches of `sequences` sequences.  bits 16: k and v are bf16
 * [sequences, kv_heads, max_len, head_dim] and the other four pointers are NULL.  bits 8 or
 * 4: k and v hold affine codes, 32-bit words [sequences, kv_heads, max_len,
 * head_dim * bits / 32] with the lowest element in the lowest bits, and each run of `group`
 * elements along the head dimension has a bf16 scale and bias
 * [sequences, kv_heads, max_len, head_dim / group]; an element is scale * code + bias (the
 * packed layout of dflash_qmm's weights).  head_dim 64, 128 or 256; group 32, 64 or 128 and
 * at most head_dim.  k and v are 16-byte aligned. */
typedef struct dflash_kv_cache {
    void* k;
    dflash_bf16* k_scales;
    dflash_bf16* k_biases;
    void* v;
    dflash_bf16* v_scales;
    dflash_bf16* v_biases;
    int sequences, kv_heads, max_len, head_dim, bits, group;
} dflash_kv_cache;

/* `lengths` (device int32 [sequences], read in stream order) is the number of tokens already
 * in each sequence's cache: its block goes to cache rows lengths[b] .. lengths[b] + tokens - 1.
 * A negative length marks a sequence that takes no part: its cache, its q_out rows and its
 * out rows are left as they were.  A length whose block would run past max_len does the same
 * and raises DFLASH_DEVERR_POSITION in the device error word. */

/* Attention prep of a batch (dflash_stack_attn_prep for several sequences and any cache).
 * qkv row r (stride ld elements) = [q (hq*d) | gate (hq*d) | k (hkv*d) | v (hkv*d)], read only.
 * q_out row r (bf16, stride ld_q; may be qkv itself with ld_q = ld) = RMSNorm (q_norm) and
 * rotary embedding of the q heads; k heads get k_norm and the rotary embedding and go, like
 * v, to the cache in its format.  Rotary position: position0 (a shared prefix's length, say)
 * + lengths[b] + t, rotate-half on the first rot dims, frequency theta^(-2i/rot), angles off
 * by at most 2^-26 + position 2^-54 of a turn.  parents (NULL, or device int32
 * [sequences, tokens], tokens <= 32): each block is a speculative tree and t becomes the
 * row's depth.  Quantisation keeps the affine rule of the weights: the edge of a group with
 * the larger magnitude is stored exactly (as a bf16 bias), the code of zero is a whole
 * number, and codes are the nearest ones under the STORED (bf16) scale and bias.  A group that
 * holds an infinity or a NaN reads back as NaN.  rot a multiple of 64 and <= d; theta > 0;
 * qkv, q_out and their row strides 16-byte aligned. */
int dflash_stack_attn_prep_batch(const dflash_bf16* qkv, long long ld, const dflash_bf16* q_norm,
                                 const dflash_bf16* k_norm, dflash_bf16* q_out, long long ld_q,
                                 const dflash_kv_cache* cache, const int32_t* lengths, int tokens, int hq, int rot,
                                 int position0, float eps, float theta, const int32_t* parents,
                                 dflash_stream_t stream);

/* Reads `rows` cache rows of every sequence back as bf16: k and v (either may be NULL) are
 * [sequences, kv_heads, rows, head_dim], row i from cache row starts[b] + i (starts NULL: i).
 * A negative start leaves its sequence's part as it was; a range past max_len does too and
 * raises DFLASH_DEVERR_POSITION.  k and v 16-byte aligned. */
int dflash_stack_kv_read(const dflash_kv_cache* cache, const int32_t* starts, int rows, dflash_bf16* k,
                         dflash_bf16* v, dflash_stream_t stream);

/* Writes `rows` bf16 rows k and v ([sequences, kv_heads, rows, head_dim], taken as they are: no
 * norm, no rotary embedding) into every sequence's cache at rows starts[b] + i (starts NULL: i),
 * quantised as dflash_stack_attn_prep_batch does.  Starts as for dflash_stack_kv_read. */
int dflash_stack_kv_write(const dflash_kv_cache* cache, const int32_t* starts, int rows, const dflash_bf16* k,
                          const dflash_bf16* v, dflash_stream_t stream);

/* After a tree round: cache row lengths[b] + rows[b * stride + i] moves to lengths[b] + i for
 * i < counts[b] (dflash_stack_kv_compact for a batch, any cache format, driven from the
 * device: rows and counts may be what dflash_accept_tree wrote as path and path_len).
 * 0 <= counts[b] <= stride <= 32 and row offsets are 0 .. 31; a sequence that breaks this or
 * would pass max_len is left as it was and raises DFLASH_DEVERR_POSITION. */
int dflash_stack_kv_compact_batch(const dflash_kv_cache* cache, const int32_t* lengths, const int32_t* rows,
                                  const int32_t* counts, int stride, dflash_stream_t stream);

/* Decode attention of a batch: token t of sequence b attends to the rows 0 .. prefix_len - 1
 * of `prefix` (one cache that every sequence shares; NULL with prefix_len 0 for none) and to
 * rows 0 .. lengths[b] + t of its own cache, or with parents (as above) to rows
 * 0 .. lengths[b] - 1 and its root-to-t path.  Head h reads kv head h / (hq / kv_heads).
 *   out[r, h d + e] = softmax(scale q K^T) V * sigmoid(gate[r, h d + e])
 * with q, gate (NULL: no gate) and out bf16 rows of hq * d elements (strides ld_q, ld_gate
 * and hq * d).  The prefix has the cache's bits, group, kv_heads and head_dim, sequences = 1.
 * Cache rows that a token does not see never reach its output, whatever they hold.  Over
 * quantised caches the operands are fp16, each row scaled by a power of two: an element under
 * 2^-11 (8 bits) or 2^-7 (4 bits) of its row's largest is held to 2^-22 or 2^-18 of that one, a
 * weight under 2^-22 of the token's largest (weight times size of its V row) to 2^-33 of that one,
 * and the rows of V that a token sees may differ in size by 2^126 (a row of zeros counts as 2^-62).
 * Over bf16 caches weights are rounded to bf16 before the product with V (not in their sum).
 * workspace: dflash_stack_attn_decode_batch_workspace_bytes() bytes of device memory, 16-byte
 * aligned, contents irrelevant before and after; calls that may run at the same time need one
 * each.  The size depends on the arguments only, not on the lengths; 0: not supported.
 * q, gate, out and their row strides 16-byte aligned. */
size_t dflash_stack_attn_decode_batch_workspace_bytes(const dflash_kv_cache* cache, int prefix_len, int tokens, int hq);
int dflash_stack_attn_decode_batch(const dflash_bf16* q, long long ld_q, const dflash_bf16* gate, long long ld_gate,
                                   const dflash_kv_cache* cache, const int32_t* lengths, const dflash_kv_cache* prefix,
                                   int prefix_len, dflash_bf16* out, int tokens, int hq, float scale,
                                   const int32_t* parents, void* workspace, size_t workspace_bytes,
                                   dflash_stream_t stream);

/* Log probabilities from rows of logits (bf16 or fp32, `vocab` values per row, row stride ld
 * elements, any alignment of the element type).  Each output may be NULL:
 *   token_logprobs fp32 [rows, n]   log softmax at tokens[row, j]; 0 for a negative token (none),
 *                                   NaN for one >= vocab
 *   entropy        fp32 [rows]      -sum p log p
 *   top_ids        int32 [rows, top], top_logprobs fp32 [rows, top]: the `top` largest logits,
 *                                   largest first, the lower id first among equals
 * Logits of -inf have probability 0.  A row that defines no distribution (a NaN or +inf in
 * it, or nothing above -inf) gives NaN throughout and ids of -1.  top <= 32 and <= vocab. */
#define DFLASH_LOGITS_BF16 0
#define DFLASH_LOGITS_FP32 1
int dflash_logprobs(const void* logits, int type, long long ld, int rows, int vocab, const int32_t* tokens, int n,
                    int top, float* token_logprobs, float* entropy, int32_t* top_ids, float* top_logprobs,
                    dflash_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* DFLASH_BATCH_H */
