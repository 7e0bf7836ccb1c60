// The choice of a kernel for attention over the 4-bit cache, and its scratch (kernels: cache4_attention.h).
#include "cache4_attention.h"

namespace we {
namespace {

constexpr size_t kScoreBytes = 256u << 20;
// workgroups that run at once: two a CU up to head dim 128, where their rings are 74 KB of its 160, one above
// (head dim 128, 16 sequences up to 4093 slots / 4 up to 65521: 512 workgroups 21.7 / 46.6 us, 768 26.5 / 51.7, 1024 30.3 / 49.9)
uint32_t slots_of(uint32_t dim) { return dim <= 128 ? 512 : 256; }

// Weights of at most 16 rows come from the scores as the attention kernel had them, 4 bytes a row and slot, instead of from a
// second pass over K with all its products; not where they would take more than kScoreBytes.
bool stored_scores(const Cache4Attention& L, uint32_t rows) {
  return rows <= 16 && (size_t)L.c.batch * L.c.kv_heads * rows * L.max_len * 4 <= kScoreBytes;
}

// rows a workgroup takes, and whether a sequence's tiles are shared out
Attn4 plan_of(const Cache4Attention& L) {
  Attn4 a{};
  a.group = L.heads / L.c.kv_heads, a.rows = L.tokens * a.group;
  a.rt = a.rows <= 16 ? 1 : most_rows((int)L.c.dim / 64);
  a.pk = a.rows <= 4 ? 4 : a.rows <= 8 ? 2 : 1;
  a.block_rows = 16 * a.rt / a.pk;
  a.row_blocks = (a.rows + a.block_rows - 1) / a.block_rows;
  const uint64_t units = (uint64_t)L.c.batch * L.c.kv_heads, blocks = units * a.row_blocks;
  // Shared out where the units alone leave half of the chip idle and a sequence may have so many tiles that a workgroup takes
  // longer over them than the second launch and the sharing do: 32 of one block of 16 rows and 128 values, fewer of more (72
  // units of 17 tiles, f32 of 64 values: 9.8 us by a workgroup each, 13.2 us in three shares; 64 units of up to 64 tiles with
  // weights: 25.9 us, 23.0 in shares; 2 units of 18 tiles of 256 values: 20.7 us, 17.0 in shares)
  const uint32_t slots = slots_of(L.c.dim);
  if (a.rows && blocks <= slots / 2 && L.c.batch <= kMostShared && (uint64_t)((L.max_len + 63) / 64) * a.rt * (L.c.dim / 64) >= 64) {
    a.split_slots = slots / a.row_blocks;
    a.split_slots = a.split_slots > units ? a.split_slots : (uint32_t)units;
  }
  return a;
}

// The scratch's parts, in order: part, ml, shares; lse; scores or operands and facts. Returns its bytes; sets the pointers when there is one.
size_t lay_out(const Cache4Attention& L, Attn4& a) {
  size_t n = 0;
  auto take = [&](size_t words) {
    float* p = L.scratch ? (float*)L.scratch + n : nullptr;
    n += (words + 3) / 4 * 4;
    return p;
  };
  const size_t rows = (size_t)L.c.batch * L.heads * L.tokens;
  if (a.split_slots) {
    const size_t shares = (size_t)a.row_blocks * a.split_slots * a.block_rows;
    a.part = take(shares * L.c.dim), a.ml = take(shares * 2), a.shares = (uint32_t*)take((size_t)L.c.batch * L.c.kv_heads * 2);
  }
  if (L.weight_out && !(a.split_slots && stored_scores(L, a.rows))) a.lse = take(rows);
  if (L.weight_out && a.rows && stored_scores(L, a.rows)) {
    a.scores = take(rows * L.max_len);
  } else if (L.weight_out && a.rows) {
    const size_t blocks = (size_t)L.c.batch * L.c.kv_heads * ((a.rows + 15) / 16);
    a.operands = (u32x4*)take(blocks * (L.c.dim / 64) * 2 * (L.dtype == F32 ? 2 : 1) * 64 * 4);
    a.facts = (RowFacts*)take(blocks * 16 * sizeof(RowFacts) / 4);
  }
  return n * 4;
}

}  // namespace

size_t cache4_attention_scratch(const Cache4Attention& L) {
  Attn4 a = plan_of(L);
  return lay_out(L, a);
}

hipError_t cache4_attention_launch(const Cache4Attention& L, hipStream_t s) {
  Attn4 a = plan_of(L);
  const uint64_t units = (uint64_t)L.c.batch * L.c.kv_heads;
  if (units > 65535 || units * a.row_blocks > 0x7fffffffull || units * ((L.max_len + 63) / 64) + units * a.rows > 0x7fffffffull)
    return hipErrorInvalidValue;
  a.kc = L.c.kc, a.ks = L.c.ks, a.vc = L.c.vc, a.vs = L.c.vs, a.q = L.q, a.out = L.out, a.counts = L.counts, a.lens = L.lens;
  a.weight = L.weight, a.weight_out = L.weight_out, a.batch = L.c.batch, a.tokens = L.tokens, a.heads = L.heads;
  a.kv_heads = L.c.kv_heads, a.capacity = L.c.capacity, a.max_len = L.max_len;
  a.q_stride = L.q_stride, a.out_stride = L.out_stride, a.causal = L.causal, a.dtype = L.dtype;
  a.scale_log2 = 1.4426950408889634f / sqrtf((float)L.c.dim);
  lay_out(L, a);
  switch (L.c.dim / 64) {
    case 1: return cache4_attention_64(a, s);
    case 2: return cache4_attention_128(a, s);
    case 3: return cache4_attention_192(a, s);
    default: return cache4_attention_256(a, s);
  }
}

}  // namespace we
