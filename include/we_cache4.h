/*
 * we_cache4.h — a key / value cache held in 4 bits, and attention over it (MI355X, gfx950).
 *
 * The part of the C ABI that decoding needs beside we.h: its contexts, buffers, streams, graphs, dtype tags, status codes
 * and messages are used here too. No counterpart in the reference, whose attention reads the K and V of one set of tokens
 * (src/kernels/attention.ts:20-51) and keeps none. Additive, like the int4 weights of we.h.
 *
 * A program appends K and V rows (after norm and RoPE, e.g. the columns of a fused QKV projection), runs attention over
 * what the cache holds, and may give up the slots that received the least attention. Lengths live on the device, so a
 * captured graph of a decode step replays with the lengths of the moment.
 */
#ifndef WE_CACHE4_H
#define WE_CACHE4_H

#include "we.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A slot holds, per kv head, a K row and a V row of `dim` values in groups of 64: a 4-bit code per value, two to a byte,
 * the first in the low bits, and per group one u32: an f16 scale (low half) and an f16 minimum (high half).
 *   value = minimum + scale * code
 * A group x is stored as: x clamped to +-65504; minimum = f16(min x); scale = f16((max x - min x) / 15);
 * code = round((x - minimum) / scale), ties to even, within 0 .. 15 (0 where scale is 0); each step rounded to f32. A NaN in
 * a group makes its scale and minimum NaN: the whole group reads as NaN. An infinity counts as +-65504.
 * `data` is one buffer of four regions, one after another: K codes u8 [batch][kv_heads][capacity][dim / 2], K scales u32
 * [batch][kv_heads][capacity][dim / 64], V codes, V scales; we_cache4_bytes bytes, 16-byte aligned. What it holds behind a
 * sequence's length is never used, whatever it is. */
#define WE_CACHE4_GROUP 64
typedef struct we_cache4 {
  uint32_t batch;    /* sequences; batch * kv_heads at most 65535 */
  uint32_t kv_heads;
  uint32_t dim;      /* a multiple of 64, at most 256 */
  uint32_t capacity; /* slots of a sequence, a multiple of 64, at most 2^24 */
  void* data;
} we_cache4;

/* Checks the shape (data may be NULL) and gives the bytes of its buffer. ctx may be NULL (we_last_error(NULL)). */
int we_cache4_bytes(we_ctx* ctx, const we_cache4* cache, uint64_t* bytes);

/* Per-sequence numbers are i32 [batch] device arrays. Values out of range are read as the nearest in range: a length as
 * 0 .. capacity, a count as 0 .. tokens. Per-slot arrays (pos i32, weight f32) are [batch][kv_heads][capacity]. An `_out`
 * array is written whole and may be the array it is computed from; apart from that, arrays and buffers that a call writes
 * must not overlap others of the call. */

/* Token i (i < counts[b], NULL: all `tokens`) of sequence b is stored in slot lens[b] + i of every kv head. Its K row is at
 * (b * tokens + i) * k_stride values of k, its V row likewise (strides 0: kv_heads * dim). dtype F32, F16 or BF16; strides
 * are multiples of 8 (F32: 4), operands 16-byte aligned. lens_out[b] = lens[b] + count; tokens that no slot is left for are
 * dropped and the length stops at the capacity. seen[b] (NULL: lens[b]) is the position of token 0: pos (may be NULL) of the
 * slot becomes seen[b] + i and seen_out[b] (NULL without seen) seen[b] + count, dropped tokens counted. weight (may be
 * NULL) of the slot becomes 0. */
int we_cache4_append(we_ctx* ctx, const we_cache4* cache, uint32_t tokens, int dtype, const void* k, uint32_t k_stride,
                     const void* v, uint32_t v_stride, const int32_t* counts, const int32_t* lens, int32_t* lens_out,
                     const int32_t* seen, int32_t* seen_out, int32_t* pos, float* weight);

/* The stored values of slots first[b] + i (first NULL: 0), i < tokens, as rows (b * tokens + i) of k and v (either may be
 * NULL), laid out and typed as we_cache4_append takes them. Rows of slots at or behind lens[b] are left as they were. */
int we_cache4_load(we_ctx* ctx, const we_cache4* cache, uint32_t tokens, const int32_t* first, const int32_t* lens, int dtype,
                   void* k, uint32_t k_stride, void* v, uint32_t v_stride);

/* Attention of `tokens` queries per sequence over its slots: query row (b * tokens + i) * q_stride of q (0: heads * dim),
 * head h against kv head h / (heads / kv_heads), softmax(q . K / sqrt(dim)) . V over the first n slots: n = lens[b], or with
 * causal lens[b] - counts[b] + i + 1 (the queries are the newest tokens, already appended). counts NULL: all `tokens`; rows
 * i >= counts[b] of out are left as they were; where n <= 0 the row is zeros. dtype F32, F16 or BF16 of q and out, strides
 * and alignment as in we_cache4_append. max_len: no length is above it (longer ones are read as max_len); 0: the capacity.
 * It sizes the launch, so a program passes what it knows.
 * weight_out (NULL: off): weight_out[b][g][slot] = weight[b][g][slot] + the sum over the queries and the heads of g of the
 * probability they gave the slot, for slots below lens[b]; others are left as they were. weight NULL: 0 + that.
 * Sums, softmax and products are f32: scores of exact 4-bit codes with q as f16 (16-bit q exactly, F32 q as two f16 values
 * that hold 22 bits, after a power of two per row); probabilities times the V scale round to f16 (F32: two f16 values). */
int we_cache4_attention(we_ctx* ctx, const we_cache4* cache, uint32_t tokens, uint32_t heads, int causal, int dtype,
                        const void* q, uint32_t q_stride, const int32_t* counts, const int32_t* lens, uint32_t max_len,
                        const float* weight, float* weight_out, void* out, uint32_t out_stride);

/* Cuts each sequence to at most `keep` slots, per kv head: lens_out[b] = min(lens[b], keep), and of the slots the
 * lens[b] - lens_out[b] lowest by (protected, weight, slot) are given up. A slot is protected if its pos is below `sinks` or
 * at least seen[b] - recent (seen NULL: lens[b]): protected slots go only when no others are left. A NaN weight counts as
 * the highest, -0 as 0. The survivors in slots from lens_out[b] on move, in order, to the slots given up below it (in
 * order); all others stay in place, so a slot's number says nothing about its age: pos does. weight_out and pos_out hold the
 * moved values in slots below lens_out[b]; others are left as they were. max_len as in we_cache4_attention. */
int we_cache4_evict(we_ctx* ctx, const we_cache4* cache, uint32_t keep, const int32_t* lens, int32_t* lens_out,
                    uint32_t max_len, const float* weight, float* weight_out, const int32_t* pos, int32_t* pos_out,
                    const int32_t* seen, uint32_t sinks, uint32_t recent);

#ifdef __cplusplus
}
#endif
#endif
