// Attention over a key / value cache held in 4 bits (include/we_cache4.h: we_cache4_attention).
//
// A row of K or V is, per group G of 64 values, mn_G + s_G u with codes u of 0 .. 15. So for a query q
//   q . K_j = sum_G s_jG (q_G . u_jG) + mn_jG sum(q_G)   and   sum_j p_j V_jG = sum_j (p_j s_jG) (u_jG - 8) + sum_j p_j (mn + 8 s)_jG
// and both products run on the codes themselves, as f16 MFMA operands, with the scales and minima applied in f32 outside:
//   * a nibble IS an f16 operand: as the low bits of an f16 it is the subnormal u 2^-24 (16 u 2^-24 from the high half of a
//     byte), which the MFMA multiplies exactly. Eight codes of K become four operand registers with four ands and a shift, and
//     no conversion; those of V, which need their sign, take four packed adds more. The factor 16 of every second code sits in
//     the other operand.
//   * S^T = K Q^T by 16x16x32 MFMAs: lane (r = lane % 16, c = lane / 16) holds, of query row r, the scores of slots
//     16 T + 4 c + i (T, i = 0 .. 3) of a tile of 64. The f32 scale and minimum of a slot meet its score there.
//   * O^T = V^T P^T: those 16 probabilities are exactly what the lane must feed as the other operand when the codes of V come
//     transposed: ds_read_b64_tr_b4 gives lane (d, c) the codes of those 16 slots for value d. P never leaves the lane.
//   * a query row is one of 16 columns, so the heads that share a kv head (and a call's few tokens) ride one pass over it.
// q is scaled by a power of two per row into f16 (16-bit q stays exact; f32 q as two f16 values, 22 bits). p s rounds to f16
// (f32: two values); its exponent is kept in range by the running maximum, which takes the largest scale of V in.
//
// A wave owns whole tiles: it streams them through its own ring in LDS by direct loads and waits for nobody until the end, when
// the workgroup's waves join their (maximum, sum, O). Long caches are split over workgroups; a second pass joins those.
//
// Bounds and figures (MI355X; head dim 128). A decode step reads 4.5 bits a value, so it is bound by HBM once it is long: 4
// sequences of up to 65521 slots, 32 / 8 heads, f16: 245 MB in 47 us with the join, 5.2 TB/s (a streaming read reaches 6.8),
// 41 us of them in the attention kernel, about 4 before the first tile is there. A short one is bound by latency: 131 slots
// 5.5 us, of which a wave's one tile takes 1.7 us and the join of the waves 0.9. A prompt is bound by the vector unit, which
// is busy 90% of the time (the MFMA 28%): 2048 queries over 8192 slots, 32 / 8 heads, f16: 379 us, 0.63 PFLOP/s.
#pragma once
#include "common.h"
#include "internal.h"

namespace we {

constexpr int NW = 4;          // waves of a workgroup
constexpr float kNone = -3e38f;  // the running maximum before the first score

struct RowFacts {
  float unit, sum[4];  // as in QRow
  uint32_t sees;       // slots; 0: no row
  uint32_t pad[2];
};
struct Attn4 {
  const uint8_t* kc;
  const uint32_t* ks;
  const uint8_t* vc;
  const uint32_t* vs;
  const void* q;
  void* out;
  const int32_t* counts;
  const int32_t* lens;
  const float* weight;
  float* weight_out;
  uint32_t batch, tokens, heads, kv_heads, group, capacity, max_len, q_stride, out_stride;
  int causal, dtype;
  float scale_log2;     // log2(e) / sqrt(dim)
  uint32_t rows;        // query rows of a kv head: tokens * group, row r = token r / group, head r % group of the kv head's
  uint32_t row_blocks;  // of block_rows rows
  uint32_t block_rows;
  uint32_t pk, rt;      // Cols, blocks of 16 rows a wave holds
  uint32_t split_slots;  // 0: one workgroup takes all of a sequence's tiles; else workgroups (of each row block) to share out
  float* part;          // shared out: O [row block][slot][block_rows][dim], times 2^-m
  float* ml;            // and (m, l) [row block][slot][block_rows][2]
  uint32_t* shares;     // and each unit's first slot and its number of shares
  float* lse;           // weights, unless they come from shared-out scores: [unit][rows], log2 of a row's sum of 2^score
  float* scores;        // weights of at most 16 rows: [unit][rows][max_len], the scores in log2 units
  u32x4* operands;      // weights of more: the rows' operands [unit][16 rows][step and plane][lane]
  RowFacts* facts;      // and the rest of them [unit][row, up to a multiple of 16]
};
hipError_t cache4_attention_64(const Attn4& a, hipStream_t s);
hipError_t cache4_attention_128(const Attn4& a, hipStream_t s);
hipError_t cache4_attention_192(const Attn4& a, hipStream_t s);
hipError_t cache4_attention_256(const Attn4& a, hipStream_t s);
// tiles of 16 query rows that a wave's registers hold
constexpr uint32_t most_rows(int ng) { return ng <= 3 ? 2 : 1; }
constexpr uint32_t kLeastTiles = 2 * NW;  // of a share
constexpr uint32_t kMostShared = 256;     // sequences of a call whose tiles are shared out

namespace {

__device__ __forceinline__ uint32_t in_range(int32_t v, uint32_t hi) { return v < 0 ? 0u : (uint32_t)v < hi ? (uint32_t)v : hi; }

// max / sum over the lanes that share a query row (r, r + 16, r + 32, r + 48)
__device__ __forceinline__ float row_max(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float row_sum(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Eight codes (a word, the first lowest) as f16 operands in the order 0 4 1 5 2 6 3 7: u 2^-24, and 16 u 2^-24 for 1 5 3 7.
__device__ __forceinline__ u32x4 codes_operand(uint32_t w) {
  const uint32_t h = w >> 8;
  return u32x4{w & 0x000f000fu, w & 0x00f000f0u, h & 0x000f000fu, h & 0x00f000f0u};
}
// The same order and factor as f16 numbers u - 8 and 16 (u - 8), exact: 1024 + u has the code in its low bits. V takes these:
// a mean over slots is small beside what its codes of one sign would sum to, and would lose that much of f32.
__device__ __forceinline__ u32x4 centred_operand(uint32_t w) {
  const uint32_t h = w >> 8;
  const f16x2 one = {(_Float16)-1032.0f, (_Float16)-1032.0f}, sixteen = {(_Float16)-1152.0f, (_Float16)-1152.0f};
  const f16x2 v0 = __builtin_bit_cast(f16x2, and_or(w, 0x000f000fu, 0x64006400u)) + one;
  const f16x2 v1 = __builtin_bit_cast(f16x2, and_or(w, 0x00f000f0u, 0x64006400u)) + sixteen;
  const f16x2 v2 = __builtin_bit_cast(f16x2, and_or(h, 0x000f000fu, 0x64006400u)) + one;
  const f16x2 v3 = __builtin_bit_cast(f16x2, and_or(h, 0x00f000f0u, 0x64006400u)) + sixteen;
  return u32x4{__builtin_bit_cast(uint32_t, v0), __builtin_bit_cast(uint32_t, v1), __builtin_bit_cast(uint32_t, v2), __builtin_bit_cast(uint32_t, v3)};
}
__device__ __forceinline__ float scale_of(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[0]; }
__device__ __forceinline__ float minimum_of(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[1]; }
// minimum + 8 scale: one instruction that reads both halves (written out, it became a conversion and a product)
__device__ __forceinline__ float middle_of(uint32_t w) {
  float r;
  asm("v_fma_mix_f32 %0, %1, %2, %1 op_sel:[0,0,1] op_sel_hi:[1,0,1]" : "=v"(r) : "v"(w), "s"(8.0f));
  return r;
}

// The 16 columns of a product hold PK * (16 / PK) query rows: with few rows (a decode step's 4 or 8 heads of a kv head) column
// t * (16 / PK) + q is row q against the t-th of PK tiles of 16 slots. The k slots of lane quarter c then belong to tile
// c / (4 / PK), and a column's operand is zero in the quarters of other tiles: each lane keeps 16 / PK scores of a 64-slot tile
// instead of 16 mostly idle ones, and the scales of those alone, for the same number of MFMAs.
template <int PK>
struct Cols {
  static constexpr int kRows = 16 / PK, kQuarters = 4 / PK, kTiles = 4 / PK;
};

// One query row of a lane as MFMA operands: for step (G, s) the 8 values of the codes word c % (4 / PK) * 2 PK + s of group
// G, in codes_operand's order and factor, times 2^e (largest value below 2^14). NP planes of f16: their sum is q.
template <int NG, int NP, int PK>
struct QRow {
  u32x4 f[NG][2 * PK][NP];
  float sum[NG];  // of 2^e q over the group, times kCode
  float unit;     // 2^-e log2(e) / sqrt(dim) / kCode: a score in log2 units is unit * (scale . dot + minimum . sum)
  static constexpr float kCode = NP == 1 ? 0x1p-24f : 1.0f;  // what a code of key_operand stands for
};

// The values of a row that a lane needs, as they are stored.
template <int NG, int NP, int PK>
struct RawRow {
  u32x4 v[NG][2 * PK * NP];
};
// `src`: the row in memory or in LDS; without `live` zeros
template <int NG, int NP, int PK>
__device__ __forceinline__ void fetch_row(bool live, const char* src, int c, RawRow<NG, NP, PK>& x) {
#pragma unroll
  for (int g = 0; g < NG; g++)
#pragma unroll
    for (int v = 0; v < 2 * PK * NP; v++) {
      x.v[g][v] = u32x4{};
      if (live) x.v[g][v] = ((const u32x4*)(src + (g * 64 + c % Cols<PK>::kQuarters * (16 * PK)) * (2 * NP)))[v];
    }
}

// F16 and BF16: their bits give the maximum, two values at a time (an infinity or a NaN
// counts as the largest finite value: it stays one in f16, in its own row); F32 below. The sums come from the operands, by
// MFMAs against ones (16 for the odd codes, which the operand holds a sixteenth of).
template <int NG, int NP, int PK>
__device__ __forceinline__ void make_row(const Attn4& a, const RawRow<NG, NP, PK>& raw, QRow<NG, NP, PK>& q) {
  constexpr int W = 8 * PK;  // words of 16-bit values a lane has of a group
  float up;
  // 2^e with the largest value 2^e in [2^13, 2^14); e in -98 .. 126, so that `unit` and 2^e are normal numbers
  auto scale = [&](uint32_t exponent, int most) {
    int e = 13 + 127 - (int)exponent;
    e = e < -98 ? -98 : e > most ? most : e;
    up = __uint_as_float((uint32_t)(e + 127) << 23);
    q.unit = __uint_as_float((uint32_t)(127 - e) << 23) * (1.0f / QRow<NG, NP, PK>::kCode) * a.scale_log2;
  };
  if constexpr (NP == 1) {
    uint32_t x[NG][W], big = 0;
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
      for (int e = 0; e < W; e++) x[g][e] = raw.v[g][e / 4][e % 4];
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 top = {};
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
      for (int e = 0; e < W; e++) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, x[g][e] & 0x7fff7fffu));
    big = top[0] > top[1] ? top[0] : top[1];
    big = __float_as_uint(row_max(__uint_as_float(big << 15))) >> 15;  // as a positive f32 of the same order, below its NaNs
    if (a.dtype == F16) {
      // at most 2^15, an f16 factor: with it every f16 is a normal number and exact
      big = big < 0x7bffu ? big : 0x7bffu;
      scale((__float_as_uint(f16_to_f32((uint16_t)big)) >> 23), 15);
      const _Float16 f = (_Float16)up;
      const f16x2 even = {f, f}, odd = even * f16x2{(_Float16)0.0625f, (_Float16)0.0625f};
#pragma unroll
      for (int g = 0; g < NG; g++)
#pragma unroll
        for (int s = 0; s < 2 * PK; s++)
#pragma unroll
          for (int j = 0; j < 4; j++) {  // operand register j: values j and j + 4
            const uint32_t lo = x[g][4 * s + j / 2], hi = x[g][4 * s + 2 + j / 2];
            const uint32_t w = __builtin_amdgcn_perm(hi, lo, j & 1 ? 0x07060302u : 0x05040100u);
            q.f[g][s][0][j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, w) * (j & 1 ? odd : even));
          }
    } else {
      big = big < 0x7f7fu ? big : 0x7f7fu;
      scale(big >> 7, 126);
      const float sixteenth = up * 0.0625f;
#pragma unroll
      for (int g = 0; g < NG; g++)
#pragma unroll
        for (int s = 0; s < 2 * PK; s++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const uint32_t lo = x[g][4 * s + j / 2], hi = x[g][4 * s + 2 + j / 2];
            if (j & 1) q.f[g][s][0][j] = pack2(__uint_as_float(lo & 0xffff0000u) * sixteenth, __uint_as_float(hi & 0xffff0000u) * sixteenth, std::true_type{});
            else q.f[g][s][0][j] = pack2(__uint_as_float(lo << 16) * up, __uint_as_float(hi << 16) * up, std::true_type{});
          }
    }
  } else {
    float x[NG][16 * PK], big = 0.0f;
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
      for (int e = 0; e < 16 * PK; e++) {
        x[g][e] = __uint_as_float(raw.v[g][e / 4][e % 4]);
        const float y = fabsf(x[g][e]);
        big = fmaxf(big, y < INFINITY ? y : 0.0f);  // an infinite or NaN value stays one in f16, in its own row
      }
    scale(__float_as_uint(row_max(big)) >> 23, 126);
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
      for (int s = 0; s < 2 * PK; s++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float f = j & 1 ? up * 0.0625f : up, p = x[g][8 * s + j] * f, r = x[g][8 * s + j + 4] * f;
          const uint32_t hi = pack2(p, r, std::true_type{});
          const f16x2 h = __builtin_bit_cast(f16x2, hi);
          q.f[g][s][0][j] = hi;
          q.f[g][s][1][j] = pack2(p - (float)h[0], r - (float)h[1], std::true_type{});
        }
  }
  const u32x4 ones = {0x3c003c00u, 0x4c004c00u, 0x3c003c00u, 0x4c004c00u};
  static_for<0, NG>([&](auto G) {
    f32x4 d = {};
    static_for<0, 2 * PK>([&](auto S) { static_for<0, NP>([&](auto P) { d = mfma_16x16x32<true>(ones, q.f[G][S][P], d); }); });
    q.sum[G] = d[0] * QRow<NG, NP, PK>::kCode;
  });
}

template <int NG, int NP>
__device__ __forceinline__ const char* q_at(const Attn4& a, uint32_t b, uint32_t gh, uint32_t i, uint32_t h) {
  return (const char*)a.q + (((size_t)b * a.tokens + i) * a.q_stride + (size_t)(gh * a.group + h) * (64 * NG)) * (2 * NP);
}

// K's operand: the codes as they are, or centred for f32 q, whose scores are worth the four adds.
template <int NP>
__device__ __forceinline__ u32x4 key_operand(uint32_t w) {
  return NP == 1 ? codes_operand(w) : centred_operand(w);
}

// The scores of a lane's four slots (codes words kw[G * 2 PK + s], scale words sw[i * NG + G] for slot i) and a query row,
// before `unit`.
template <int NG, int NP, int PK>
__device__ __forceinline__ f32x4 scores(const uint32_t (&kw)[2 * PK * NG], const uint32_t (&sw)[4 * NG], const QRow<NG, NP, PK>& q, float zero) {
  f32x4 s;
  static_for<0, NG>([&](auto G) {
    f32x4 d = {};
    static_for<0, 2 * PK>([&](auto S) {
      const u32x4 k = key_operand<NP>(kw[G * 2 * PK + S]);
      static_for<0, NP>([&](auto P) { d = mfma_16x16x32<true>(k, q.f[G][S][P], d); });
    });
    static_for<0, 4>([&](auto I) {
      const uint32_t w = sw[I * NG + G];
      const float m = __builtin_fmaf(NP == 1 ? minimum_of(w) : middle_of(w), q.sum[G], G == 0 ? zero : s[I()]);
      s[I()] = __builtin_fmaf(scale_of(w), d[I()], m);
    });
  });
  return s;
}

__device__ __forceinline__ void unit_of(const Attn4& a, uint32_t unit, uint32_t& len, uint32_t& count) {
  const uint32_t b = unit / a.kv_heads;
  len = in_range(a.lens[b], a.max_len);
  count = a.counts ? in_range(a.counts[b], a.tokens) : a.tokens;
}
// How the tiles of all sequences are shared out: `chunk` tiles a workgroup, near the least (and no fewer than kLeastTiles) with
// which the shares of all kv heads fit the slots. Lengths are on the device only, so every workgroup works it out, its lanes
// a sequence each (at most kMostShared). A sequence without slots has one share, which writes its rows. Shares are numbered
// sequence by sequence, kv head by kv head.
__device__ __forceinline__ uint32_t prefix_sum(uint32_t x) {  // inclusive, over the lanes
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false);  // from the lanes 1, 2, 4, 8 before, in rows of 16
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false);  // the last of row 0 and 2 to row 1 and 3
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false);  // the last of row 1 to rows 2 and 3
  return x;
}
__device__ __forceinline__ uint32_t last_lane(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)x, 63); }

struct Share {
  uint32_t unit, first, count, index, chunk;  // share `index` of the unit's `count`, which start at slot `first`
};
// the slot's share; false: it has none
__device__ __forceinline__ bool share_of(const Attn4& a, uint32_t slot, Share& out) {
  constexpr int N = kMostShared / 64;
  const uint32_t lane = threadIdx.x & 63;
  uint32_t tiles[N], n[N], all = 0;
#pragma unroll
  for (int k = 0; k < N; k++) {
    tiles[k] = 0;
    if (64u * k < a.batch) {
      if (64 * k + lane < a.batch) tiles[k] = (in_range(a.lens[64 * k + lane], a.max_len) + 63) / 64;
      all += last_lane(prefix_sum(tiles[k]));
    }
  }
  // (products of f32 here only choose among chunks that are all right; the share counts are exact)
  const float per = (float)a.kv_heads * __builtin_amdgcn_rcpf((float)a.split_slots);
  uint32_t chunk = (uint32_t)((float)all * per) + 1;
  chunk = chunk > kLeastTiles ? chunk : kLeastTiles;
  for (;;) {  // ends: with a chunk of the longest sequence there are as many shares as units, and the slots are no fewer
    const float inv = __builtin_amdgcn_rcpf((float)chunk);
    all = 0;
#pragma unroll
    for (int k = 0; k < N; k++) {
      if (64u * k < a.batch) {
        uint32_t q = (uint32_t)((float)tiles[k] * inv);  // within one of the quotient
        while (q * chunk < tiles[k]) q++;
        while (q && (q - 1) * chunk >= tiles[k]) q--;
        n[k] = 64 * k + lane < a.batch ? (q ? q : 1) : 0;
        all += last_lane(prefix_sum(n[k]));
      }
    }
    if (all * a.kv_heads <= a.split_slots) break;
    chunk += (uint32_t)((float)chunk * ((float)all * per - 1.0f) * 0.5f) + 1;  // half of what is too much
  }
  uint32_t before = 0;
#pragma unroll
  for (int k = 0; k < N; k++) {
    if (64u * k < a.batch) {
      const uint32_t to = prefix_sum(n[k]), sum = last_lane(to);
      const uint64_t past = __ballot((before + to) * a.kv_heads > slot);
      if (past) {
        const int b = __builtin_ctzll(past);
        const uint32_t c = (uint32_t)__builtin_amdgcn_readlane((int)n[k], b);
        const uint32_t base = (before + (uint32_t)__builtin_amdgcn_readlane((int)to, b) - c) * a.kv_heads, head = (slot - base) / c;
        out = Share{(64 * k + b) * a.kv_heads + head, base + head * c, c, slot - base - head * c, chunk};
        return true;
      }
      before += sum;
    }
  }
  return false;
}

// the slots that token i sees
__device__ __forceinline__ uint32_t sees(const Attn4& a, uint32_t len, uint32_t count, uint32_t i) {
  const int32_t n = a.causal ? (int32_t)(len + i + 1) - (int32_t)count : (int32_t)len;
  return n < 0 ? 0u : (uint32_t)n;
}

__device__ __forceinline__ void store_row(const Attn4& a, size_t at, f32x4 v) {
  if (a.dtype == F32) *(f32x4*)((float*)a.out + at) = v;
  else if (a.dtype == F16) *(u32x2*)((uint16_t*)a.out + at) = u32x2{pack2(v[0], v[1], std::true_type{}), pack2(v[2], v[3], std::true_type{})};
  else *(u32x2*)((uint16_t*)a.out + at) = u32x2{pack2(v[0], v[1], std::false_type{}), pack2(v[2], v[3], std::false_type{})};
}

// 16 bytes a lane from an address of its own straight to LDS, lane i to dst + 16 i (dma16s with a 64-bit address)
__device__ __forceinline__ void dma16g(const char* src, void* dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"((uint32_t)(uintptr_t)(lds_ptr_t*)dst), "v"(src)
               : "memory");
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// A stage of a wave's ring: 64 slots as K codes and V codes [tile of 16][16-byte piece][16 slots] and K and V scale words in slot
// order.
template <int NG>
struct Ring {
  static constexpr int kCodes = 2048 * NG, kScales = 256 * NG, kBytes = 2 * (kCodes + kScales), kStages = 2;
  static constexpr int kLoads = 4 * NG + 2;
  template <int NP, int PK>
  static constexpr int kQLoads = (16 / PK * 8 * NG * NP + 63) / 64;  // of the rows of q
};

// RT blocks of 16 rows (PK 1), or 16 / PK rows (RT 1). Two blocks at two waves a SIMD (256 registers): what a tile's codes cost
// is shared by both (2048 queries over 8192 slots: two blocks at one wave 650 us, at two 420). Three or four blocks do not fit.
template <int NG, int RT, int NP, int PK>
__global__ void __launch_bounds__(64 * NW, NG <= 2 ? 2 : 1) cache4_attention_kernel(Attn4 a) {
  using R = Ring<NG>;
  using C = Cols<PK>;
  static_assert(RT == 1 || PK == 1, "blocks of rows are whole");
  constexpr int DIM = 64 * NG, ROW = DIM + 4;  // floats of a joined row in LDS, padded against bank conflicts
  static_assert(NW * 16 * ROW * 4 + NW * 16 * 8 <= NW * R::kStages * R::kBytes, "the join fits the ring");
  constexpr uint32_t ROWS = RT * C::kRows;
  constexpr bool ONCE = PK > 1 || (RT == 1 && most_rows(NG) > 1);  // one row block: no other workgroup reads these slots
  constexpr int kPieces = 8 * NG * NP;  // of 16 bytes, of a row of q
  __shared__ __attribute__((aligned(1024))) char lds[NW * R::kStages * R::kBytes + (RT == 1 ? R::template kQLoads<NP, PK> * 1024 : 0)];
  char* lds_q = lds + NW * R::kStages * R::kBytes;
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int rt = r / C::kRows, cs = c / C::kQuarters;  // the column's tile, the quarter's
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // (unit, split, row block): each XCD takes a run of blocks of one unit, so that the row blocks that read its slots share an
  // L2; the last row blocks first, which see the most
  uint32_t id = blockIdx.x;
  if ((gridDim.x & 7u) == 0u) id = (id & 7u) * (gridDim.x >> 3) + (id >> 3);
  const uint32_t rb = a.row_blocks - 1 - id % a.row_blocks, slot = id / a.row_blocks;
  uint32_t unit = slot, t0 = 0, chunk = ~0u;
  if (a.split_slots) {
    Share sh;
    if (!share_of(a, slot, sh)) return;
    unit = (uint32_t)__builtin_amdgcn_readfirstlane((int)sh.unit);
    t0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)(sh.index * sh.chunk));
    chunk = sh.chunk;
    if (rb == 0 && sh.index == 0 && threadIdx.x == 0) a.shares[unit * 2] = sh.first, a.shares[unit * 2 + 1] = sh.count;
  }
  uint32_t len, count;
  unit_of(a, unit, len, count);
  const uint32_t b = unit / a.kv_heads, gh = unit % a.kv_heads;
  const uint32_t row0 = rb * ROWS, rows = count * a.group;
  if (row0 >= rows) return;
  const uint32_t last = row0 + ROWS < rows ? row0 + ROWS - 1 : rows - 1;
  const uint32_t most = sees(a, len, count, last / a.group), least = sees(a, len, count, row0 / a.group);
  uint32_t t1 = (most + 63) / 64;
  t1 = t1 > t0 && t1 - t0 > chunk ? t0 + chunk : t1;

  const size_t slots = (size_t)unit * a.capacity;
  const __amdgpu_buffer_rsrc_t rkc = __builtin_amdgcn_make_buffer_rsrc((void*)(a.kc + slots * (32 * NG)), (short)0, (int)(a.capacity * (32 * NG)), 0x00020000);
  const __amdgpu_buffer_rsrc_t rvc = __builtin_amdgcn_make_buffer_rsrc((void*)(a.vc + slots * (32 * NG)), (short)0, (int)(a.capacity * (32 * NG)), 0x00020000);
  const __amdgpu_buffer_rsrc_t rks = __builtin_amdgcn_make_buffer_rsrc((void*)(a.ks + slots * NG), (short)0, (int)(a.capacity * (4 * NG)), 0x00020000);
  const __amdgpu_buffer_rsrc_t rvs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.vs + slots * NG), (short)0, (int)(a.capacity * (4 * NG)), 0x00020000);
  char* ring = lds + wave * (R::kStages * R::kBytes);
  auto issue = [&](uint32_t t, int stage) {
    char* to = ring + stage * R::kBytes;
    static_for<0, 2 * NG>([&](auto J) {
      const uint32_t tc = J * 4 + c, o = (16 * (tc / (2 * NG)) + r) * (32 * NG) + tc % (2 * NG) * 16;
      dma16s<ONCE>(rkc, to + J * 1024, o, t * (2048 * NG));
      dma16s<ONCE>(rvc, to + R::kCodes + J * 1024, o, t * (2048 * NG));
    });
    if (lane < 16 * NG) {
      dma16s<ONCE>(rks, to + 2 * R::kCodes, lane * 16, t * (256 * NG));
      dma16s<ONCE>(rvs, to + 2 * R::kCodes + R::kScales, lane * 16, t * (256 * NG));
    }
  };
  t1 = (uint32_t)__builtin_amdgcn_readfirstlane((int)t1);
  uint32_t t = t0 + wave;
  QRow<NG, NP, PK> q[RT];
  uint32_t vis[RT];
  float m[RT], le[RT], lo[RT], me[RT][NG], mo[RT][NG];  // l and the sum of p (minimum + 8 scale): over even slots i, and odd ones / 16
  f32x4 o[RT][4 * NG];
  // The rows of q come first, and with one block of them through LDS (every wave brings all of them to the same place): the
  // compiler knows nothing of the direct loads and would wait for all of them before it took a register load's result.
  if constexpr (RT == 1) {
    static_for<0, R::template kQLoads<NP, PK>>([&](auto J) {
      const uint32_t p = J * 64 + lane, row = row0 + p / kPieces;
      if (p < C::kRows * kPieces && row < rows) dma16g(q_at<NG, NP>(a, b, gh, row / a.group, row % a.group) + p % kPieces * 16, lds_q + J * 1024);
    });
    if (t < t1) issue(t, 0);
    if (t + NW < t1) issue(t + NW, 1);
    if (t + NW < t1) wait_loads<2 * R::kLoads>();
    else if (t < t1) wait_loads<R::kLoads>();
    else wait_loads<0>();
  }
  static_for<0, RT>([&](auto I) {
    const uint32_t row = row0 + 16 * I + r % C::kRows;
    const bool live = row < rows;
    const uint32_t i = live ? row / a.group : 0, h = live ? row % a.group : 0;
    const char* src = RT == 1 ? lds_q + r % C::kRows * (kPieces * 16) : q_at<NG, NP>(a, b, gh, i, h);
    RawRow<NG, NP, PK> raw;
    fetch_row<NG, NP, PK>(live && rt == cs, src, c, raw);
    make_row<NG, NP, PK>(a, raw, q[I]);
    vis[I] = live ? sees(a, len, count, i) : len;
    m[I] = kNone, le[I] = lo[I] = 0.0f;
    static_for<0, NG>([&](auto G) { me[I][G] = mo[I][G] = 0.0f; });
    static_for<0, 4 * NG>([&](auto D) { o[I][D] = f32x4{}; });
  });
  if (RT > 1 && t < t1) issue(t, 0);
  if (RT > 1 && t + NW < t1) issue(t + NW, 1);
  float zero = 0.0f;
  asm("" : "+v"(zero));  // a product of a scale is one instruction when it adds something

  uint32_t slim = 0;   // the largest V scale seen, as f16 bits, rounded up to below a power of two
  float bound = -14.0f;  // log2 of that power
  auto tile = [&](uint32_t t, const char* st, auto MASK) {
    const uint32_t k0 = t * 64 + 16 * rt + 4 * c;  // the lane's slots: k0 + 16 PK X + i
    f32x4 s[RT][C::kTiles];
    static_for<0, C::kTiles>([&](auto X) {
      uint32_t kw[2 * PK * NG], sw[4 * NG];
      static_for<0, NG>([&](auto G) {
        // words c % (4 / PK) * 2 PK .. of the group's 8: two, or one or two pieces of four
        const char* at = st + ((PK * X + cs) * (2 * NG) + 2 * G) * 256 + r * 16;
        if constexpr (PK == 1) {
          const u32x2 w = *(const u32x2*)(at + (c / 2) * 256 + c % 2 * 8);
          kw[2 * G] = w.x, kw[2 * G + 1] = w.y;
        } else {
          static_for<0, PK / 2>([&](auto V) {
            const u32x4 w = *(const u32x4*)(at + (c % C::kQuarters + V) * 256);
            static_for<0, 4>([&](auto E) { kw[2 * PK * G + 4 * V + E] = w[E()]; });
          });
        }
        const u32x4 v = *(const u32x4*)(st + 2 * R::kCodes + (16 * (PK * X + rt) + 4 * c) * (4 * NG) + G * 16);
        static_for<0, 4>([&](auto E) { sw[4 * G + E] = v[E()]; });
      });
      if constexpr (RT == 1) {
        s[0][X] = scores<NG, NP, PK>(kw, sw, q[0], zero);
      } else {
        static_for<0, RT>([&](auto I) { s[I][X] = scores<NG, NP, PK>(kw, sw, q[I], zero); });
      }
    });
    if constexpr (RT == 1) {
      if (a.scores && r % C::kRows < rows) {
        float* to = a.scores + ((size_t)unit * a.rows + r % C::kRows) * a.max_len + k0;
        static_for<0, C::kTiles>([&](auto X) {
          if (!MASK || k0 + 16 * PK * X + 4 <= a.max_len) {
            *(f32x4*)(to + 16 * PK * X) = s[0][X] * q[0].unit;
          } else {
            static_for<0, 4>([&](auto E) { if (k0 + 16 * PK * X + E < a.max_len) to[16 * PK * X + E] = s[0][X][E()] * q[0].unit; });
          }
        });
      }
    }
    float mx[RT];
    bool high = false;
    static_for<0, RT>([&](auto I) {
      static_for<0, C::kTiles>([&](auto X) {
        static_for<0, 4>([&](auto E) {
          if constexpr (MASK) s[I][X][E()] = k0 + 16 * PK * X + E < vis[I] ? s[I][X][E()] : -INFINITY;
          mx[I] = X + E == 0 ? s[I][0][0] : fmaxf(mx[I], s[I][X][E()]);
        });
      });
      mx[I] *= q[I].unit;
      high |= mx[I] + bound > m[I] + 15.0f;
    });
    uint32_t sc = 0;
    static_for<0, NG>([&](auto G) {
      uint32_t w = *(const uint32_t*)(st + 2 * R::kCodes + R::kScales + (lane + 64 * G) * 4) & 0xffffu;
      w = w < 0x7c00u ? w : 0u;  // a NaN's rows are NaN anyway; the others' range is not its
      if constexpr (MASK) sc = max(sc, t * 64 + (lane + 64 * G) / NG < most ? w : 0u);
      else sc = max(sc, w);
    });
    // p s stays below 2^16: the running maximum (a whole number: of a row's scores, plus the scales' bound, less 7) moves when
    // a score would pass it by 15
    if (__builtin_expect(__any(high || sc > slim), 0)) {
      for (int x = 1; x < 64; x *= 2) sc = max(sc, (uint32_t)__shfl_xor((int)sc, x));
      slim = max(slim, (uint32_t)__builtin_amdgcn_readfirstlane(sc) | 0x3ffu);
      bound = fmaxf((float)(slim >> 10) - 14.0f, -14.0f);
      static_for<0, RT>([&](auto I) {
        const float to = fmaxf(m[I], ceilf(row_max(mx[I])) + bound - 7.0f), f = __builtin_amdgcn_exp2f(m[I] - to);
        m[I] = to, le[I] *= f, lo[I] *= f;
        static_for<0, NG>([&](auto G) { me[I][G] *= f, mo[I][G] *= f; });
        static_for<0, 4 * NG>([&](auto D) { o[I][D] *= f; });
      });
    }
    const float up = NP == 1 ? 1.0f : __builtin_amdgcn_exp2f(7.0f - bound);
    static_for<0, RT>([&](auto I) {
      // the odd codes of V are 16 times too large. F32: the offset that keeps p s in range is a factor and not part of the
      // exponent, whose rounding grows with it.
      const float off = NP == 1 ? 0.0f : 7.0f - bound, even = m[I] + off, odd = NP == 1 ? m[I] + 4.0f : even;
      static_for<0, C::kTiles>([&](auto X) {
        static_for<0, 4>([&](auto E) {
          s[I][X][E()] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[I][X][E()], q[I].unit, -(E & 1 ? odd : even)));
          if constexpr (NP == 2) s[I][X][E()] *= E & 1 ? up * 0.0625f : up;
          if constexpr (E & 1) lo[I] += s[I][X][E()];
          else le[I] += s[I][X][E()];
        });
      });
    });
    uint32_t vw[C::kTiles][4 * NG];
    static_for<0, C::kTiles>([&](auto X) {
      static_for<0, NG>([&](auto G) {
        const u32x4 v = *(const u32x4*)(st + 2 * R::kCodes + R::kScales + (16 * (PK * X + rt) + 4 * c) * (4 * NG) + G * 16);
        static_for<0, 4>([&](auto E) { vw[X][4 * G + E] = v[E()]; });
      });
    });
    const char* vt = st + R::kCodes + ((r / 4) * (2 * NG * 16) + 4 * c + r % 4) * 16;
    static_for<0, NG>([&](auto G) {
      // operand register i of product K: slots i of tiles 2 K and 2 K + 1
      u32x4 pf[RT][2][NP];
      static_for<0, RT>([&](auto I) {
        // p s of the lane's slot i of tile X, with p's part of the minima
        auto weighted = [&](auto X, auto E) {
          const float p = s[I][X][E()];
          uint32_t w = vw[X][E * NG + G];
          if constexpr (MASK) w = k0 + 16 * PK * X + E < vis[I] ? w : 0u;  // p is 0 there; the scale may be anything
          float& mn = E & 1 ? mo[I][G] : me[I][G];
          mn = __builtin_fmaf(p, middle_of(w), mn);
          return __builtin_fmaf(p, scale_of(w), zero);
        };
        static_for<0, 4>([&](auto E) {
          if constexpr (PK == 1) {
            static_for<0, 2>([&](auto K) {
              const float p0 = weighted(std::integral_constant<int, 2 * K>{}, E), p1 = weighted(std::integral_constant<int, 2 * K + 1>{}, E);
              const f16x2 h = {(_Float16)p0, (_Float16)p1};
              pf[I][K][0][E()] = __builtin_bit_cast(uint32_t, h);
              if constexpr (NP == 2) pf[I][K][1][E()] = pack2(p0 - (float)h[0], p1 - (float)h[1], std::true_type{});
            });
          } else {
            static_for<0, C::kTiles>([&](auto X) {
              const float ps = weighted(X, E);
              uint32_t h[NP];
              h[0] = f32_to_f16(ps);
              if constexpr (NP == 2) h[1] = f32_to_f16(ps - f16_to_f32((uint16_t)h[0]));
              static_for<0, NP>([&](auto P) {
                const uint32_t v = h[P] << (16 * (rt & 1));
                if constexpr (PK == 2) {
                  pf[I][X][P][E()] = v;
                } else {
                  pf[I][0][P][E()] = rt < 2 ? v : 0u;
                  pf[I][1][P][E()] = rt < 2 ? 0u : v;
                }
              });
            });
          }
        });
      });
      static_for<0, 4>([&](auto D) {
        typedef int v2i __attribute__((ext_vector_type(2)));
        const char* at = vt + (2 * G + D / 2) * 256 + D % 2 * 8;
        const v2i w = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) v2i*)at);
        const u32x4 v0 = centred_operand((uint32_t)w.x), v1 = centred_operand((uint32_t)w.y);
        static_for<0, RT>([&](auto I) {
          static_for<0, NP>([&](auto P) {
            o[I][4 * G + D] = mfma_16x16x32<true>(v0, pf[I][0][P], o[I][4 * G + D]);
            o[I][4 * G + D] = mfma_16x16x32<true>(v1, pf[I][1][P], o[I][4 * G + D]);
          });
        });
      });
    });
  };

  // the tiles that every row sees whole, then those at the rows' ends
  int stage = 0;
  auto step = [&](auto MASK) {
    if (t + NW < t1) wait_loads<R::kLoads>();
    else wait_loads<0>();
    tile(t, ring + stage * R::kBytes, MASK);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage's reads are done before it is filled again
    if (t + 2 * NW < t1) issue(t + 2 * NW, stage);
    t += NW, stage ^= 1;
  };
  const uint32_t whole = t1 < least / 64 ? t1 : least / 64;
  while (t < whole) step(std::false_type{});
  while (t < t1) step(std::true_type{});

  // join the waves, and a row's PK columns: the largest maximum, all sums brought to it, their total
  float* ml = (float*)lds;           // [wave][16][2]
  float* joined = ml + NW * 16 * 2;  // [wave][16][ROW]
  static_for<0, RT>([&](auto I) {
    const float l = row_sum(le[I] + 16.0f * lo[I]);
    __syncthreads();
    if (c == 0) ml[(wave * 16 + r) * 2] = m[I], ml[(wave * 16 + r) * 2 + 1] = l;
    static_for<0, NG>([&](auto G) {
      const float mn = row_sum(me[I][G] + 16.0f * mo[I][G]);
      static_for<0, 4>([&](auto D) { *(f32x4*)(joined + (wave * 16 + r) * ROW + (4 * G + D) * 16 + 4 * c) = o[I][4 * G + D] + mn; });
    });
    __syncthreads();
    for (uint32_t x = threadIdx.x; x < C::kRows * DIM / 4; x += 64 * NW) {
      const uint32_t rr = x / (DIM / 4), d = x % (DIM / 4) * 4, row = row0 + 16 * I + rr;
      if (row >= rows) continue;
      float mm = kNone, ll = 0.0f;
#pragma unroll
      for (int w = 0; w < NW * PK; w++) mm = fmaxf(mm, ml[(w * C::kRows + rr) * 2]);
      f32x4 v = {};
#pragma unroll
      for (int w = 0; w < NW * PK; w++) {
        const float f = __builtin_amdgcn_exp2f(ml[(w * C::kRows + rr) * 2] - mm);
        ll = __builtin_fmaf(f, ml[(w * C::kRows + rr) * 2 + 1], ll);
        v += f * *(const f32x4*)(joined + (w * C::kRows + rr) * ROW + d);
      }
      if (a.split_slots) {
        const size_t at = ((size_t)rb * a.split_slots + slot) * ROWS + 16 * I + rr;
        *(f32x4*)(a.part + at * DIM + d) = v;
        if (d == 0) a.ml[at * 2] = mm, a.ml[at * 2 + 1] = ll;
        continue;
      }
      if (a.lse && d == 0) a.lse[(size_t)unit * a.rows + row] = mm + __builtin_amdgcn_logf(ll);
      const float inv = ll != 0.0f ? 1.0f / ll : 0.0f;  // 0: a row that sees nothing
      const size_t at = ((size_t)b * a.tokens + row / a.group) * a.out_stride + (size_t)(gh * a.group + row % a.group) * DIM + d;
      store_row(a, at, v * inv);
    }
  });
}

// The shares of a row joined by one workgroup (bound by latency: 128 rows of 16 shares 4.5 us): DIM / 4 threads a share,
// several shares at once, brought to the largest maximum and summed in a fixed order.
template <int NG>
__device__ __forceinline__ void join_row(const Attn4& a, uint32_t ur) {
  constexpr int DIM = 64 * NG, LANES = DIM / 4, SIDE = 64 * NW / LANES;
  __shared__ f32x4 sums[SIDE][LANES];
  const uint32_t unit = ur / a.rows, row = ur % a.rows;
  const uint32_t first = a.shares[unit * 2], n = a.shares[unit * 2 + 1];
  uint32_t len, count;
  unit_of(a, unit, len, count);
  if (row >= count * a.group) return;
  const size_t at = ((size_t)(row / a.block_rows) * a.split_slots + first) * a.block_rows + row % a.block_rows;
  const uint32_t lane = threadIdx.x & 63;
  float top = kNone, l = 0.0f;
  for (uint32_t s = lane; s < n; s += 64) top = fmaxf(top, a.ml[(at + (size_t)s * a.block_rows) * 2]);
#pragma unroll
  for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
  for (uint32_t s = lane; s < n; s += 64) {
    const float* ml = a.ml + (at + (size_t)s * a.block_rows) * 2;
    l += ml[1] * __builtin_amdgcn_exp2f(ml[0] - top);
  }
#pragma unroll
  for (int x = 1; x < 64; x *= 2) l += __shfl_xor(l, x);
  const uint32_t side = threadIdx.x / LANES, d = threadIdx.x % LANES;
  f32x4 v = {};
  if (side < SIDE) {
    for (uint32_t s = side; s < n; s += SIDE) {
      const size_t x = at + (size_t)s * a.block_rows;
      v += __builtin_amdgcn_exp2f(a.ml[x * 2] - top) * *(const f32x4*)(a.part + x * DIM + d * 4);
    }
    sums[side][d] = v;
  }
  __syncthreads();
  if (side) return;
  if (a.lse && threadIdx.x == 0) a.lse[ur] = top + __builtin_amdgcn_logf(l);
#pragma unroll
  for (int x = 1; x < SIDE; x++) v += sums[x][d];
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  const size_t to = ((size_t)(unit / a.kv_heads) * a.tokens + row / a.group) * a.out_stride +
                    (size_t)(unit % a.kv_heads * a.group + row % a.group) * DIM + d * 4;
  store_row(a, to, v * inv);
}

// log2 of a row's sum of 2^score; the lanes that share the row take a share in four each
__device__ __forceinline__ float row_lse(const Attn4& a, uint32_t unit, uint32_t row, int c) {
  if (!a.split_slots) return a.lse[(size_t)unit * a.rows + row];
  const uint32_t first = a.shares[unit * 2], n = a.shares[unit * 2 + 1];
  const float* ml = a.ml + (((size_t)(row / a.block_rows) * a.split_slots + first) * a.block_rows + row % a.block_rows) * 2;
  float top = kNone, l = 0.0f;
  for (uint32_t s = c; s < n; s += 4) top = fmaxf(top, ml[(size_t)s * a.block_rows * 2]);
  top = row_max(top);
  for (uint32_t s = c; s < n; s += 4) l += ml[(size_t)s * a.block_rows * 2 + 1] * __builtin_amdgcn_exp2f(ml[(size_t)s * a.block_rows * 2] - top);
  return top + __builtin_amdgcn_logf(row_sum(l));
}

// The attention each slot received, from the stored scores of at most 16 rows: a thread takes four slots. (16 sequences of up
// to 4093 slots, 28 / 4 heads: 6.7 us with the joins; from K again, with all its products, 12.)
__device__ __forceinline__ void receive_scores(const Attn4& a, uint32_t unit, uint32_t block) {
  __shared__ float lse[16];
  uint32_t len, count;
  unit_of(a, unit, len, count);
  const uint32_t rows = count * a.group, k = (block * 64 * NW + threadIdx.x) * 4;
  if (block * 64 * NW * 4 >= len) return;
  f32x4 v[8];
  auto fetch = [&](uint32_t r0) {
#pragma unroll
    for (int x = 0; x < 8; x++) {
      const float* s = a.scores + ((size_t)unit * a.rows + r0 + x) * a.max_len + k;
      v[x] = f32x4{};
      if (r0 + x >= rows || k >= len) continue;
      if (a.max_len % 4 == 0) {  // rows of scores are 16-byte aligned
        v[x] = *(const f32x4*)s;
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) v[x][e] = k + e < a.max_len ? s[e] : 0.0f;
      }
    }
  };
  fetch(0);
  if (rows && threadIdx.x < 64) {
    const uint32_t r = threadIdx.x & 15;
    const float v = row_lse(a, unit, r < rows ? r : 0, (int)(threadIdx.x >> 4));
    if (threadIdx.x < 16) lse[r] = v;
  }
  __syncthreads();
  if (k >= len) return;
  f32x4 sum = {};
  for (uint32_t r0 = 0; r0 < rows; r0 += 8) {
    if (r0) fetch(r0);
#pragma unroll
    for (int x = 0; x < 8; x++) {
      if (r0 + x >= rows) break;
      const uint32_t vis = sees(a, len, count, (r0 + x) / a.group);
#pragma unroll
      for (int e = 0; e < 4; e++) sum[e] += k + e < vis ? __builtin_amdgcn_exp2f(v[x][e] - lse[r0 + x]) : 0.0f;
    }
  }
  const size_t slot = (size_t)unit * a.capacity + k;
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (k + e < len) a.weight_out[slot + e] = (a.weight ? a.weight[slot + e] : 0.0f) + sum[e];
}

// The operands of 16 rows for `receive`, by a wave. (Written by the attention kernel, they cost its loop more in registers, 2048
// queries over 8192 slots 380 -> 405 us, than this takes.)
template <int NG, int NP>
__device__ __forceinline__ void keep_operands(const Attn4& a, uint32_t block) {
  const uint32_t blocks = (a.rows + 15) / 16, unit = block / blocks, row0 = block % blocks * 16;
  if (unit >= a.batch * a.kv_heads) return;
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  uint32_t len, count;
  unit_of(a, unit, len, count);
  const uint32_t row = row0 + r, rows = count * a.group;
  if (row0 >= rows) return;
  const bool live = row < rows;
  const uint32_t i = live ? row / a.group : 0, h = live ? row % a.group : 0;
  RawRow<NG, NP, 1> raw;
  QRow<NG, NP, 1> q;
  fetch_row<NG, NP, 1>(live, q_at<NG, NP>(a, unit / a.kv_heads, unit % a.kv_heads, i, h), c, raw);
  make_row<NG, NP, 1>(a, raw, q);
  static_for<0, NG>([&](auto G) {
    static_for<0, 2>([&](auto S) {
      static_for<0, NP>([&](auto P) { a.operands[(((size_t)block * NG + G) * 2 * NP + S * NP + P) * 64 + lane] = q.f[G][S][P]; });
    });
  });
  if (c) return;
  RowFacts f{};
  f.unit = q.unit, f.sees = live ? sees(a, len, count, i) : 0;
  static_for<0, NG>([&](auto G) { f.sum[G] = q.sum[G]; });
  a.facts[(size_t)block * 16 + r] = f;
}

// The attention each slot received, from the cache: a workgroup takes 64 slots and its waves the query rows, every NW-th
// 16 each, as operands, with their sums known and the next 16 on their way. No slot is written by two workgroups, and the rows are added in
// one order. Bound by the vector unit: 3563 rows over 2 x 4099 slots, 4 kv heads 53 us.
template <int NG, int NP>
__device__ __forceinline__ void receive(const Attn4& a, uint32_t unit, uint32_t tile) {
  __shared__ float sums[NW][64];
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t len, count;
  unit_of(a, unit, len, count);
  const uint32_t k0 = tile * 64;
  if (k0 >= len) return;
  const size_t slot = (size_t)unit * a.capacity + k0;
  uint32_t kw[4][2 * NG], sw[4][4 * NG];
  static_for<0, 4>([&](auto T) {
    static_for<0, NG>([&](auto G) {
      const u32x2 w = *(const u32x2*)(a.kc + (slot + 16 * T + r) * (32 * NG) + G * 32 + c * 8);
      kw[T][2 * G] = w.x, kw[T][2 * G + 1] = w.y;
      const u32x4 v = *(const u32x4*)(a.ks + (slot + 16 * T + 4 * c) * NG + G * 4);
      static_for<0, 4>([&](auto E) { sw[T][4 * G + E] = v[E()]; });
    });
  });
  const uint32_t rows = count * a.group;
  // the first row that sees a slot of the tile
  const uint32_t from = a.causal && k0 + count > len ? (k0 + count - len) * a.group : 0;
  float sum[16], zero = 0.0f;
  asm("" : "+v"(zero));
  for (int x = 0; x < 16; x++) sum[x] = 0.0f;
  QRow<NG, NP, 1> next;
  float lse = 0.0f;
  uint32_t vis = 0;
  auto fetch = [&](uint32_t row0) {
    const size_t block = (size_t)unit * ((a.rows + 15) / 16) + row0 / 16;
    static_for<0, NG>([&](auto G) {
      static_for<0, 2>([&](auto S) {
        static_for<0, NP>([&](auto P) { next.f[G][S][P] = a.operands[((block * NG + G) * 2 * NP + S * NP + P) * 64 + lane]; });
      });
    });
    const RowFacts f = a.facts[block * 16 + r];
    next.unit = f.unit, vis = f.sees;
    static_for<0, NG>([&](auto G) { next.sum[G] = f.sum[G]; });
    lse = a.lse[(size_t)unit * a.rows + (row0 + r < rows ? row0 + r : 0)];
  };
  uint32_t row0 = from / 16 * 16 + wave * 16;
  if (row0 < rows) fetch(row0);
  for (; row0 < rows; row0 += 16 * NW) {
    const QRow<NG, NP, 1> q = next;
    const uint32_t end = vis;
    const float sub = lse;
    if (row0 + 16 * NW < rows) fetch(row0 + 16 * NW);
    static_for<0, 4>([&](auto T) {
      const f32x4 s = scores<NG, NP, 1>(kw[T], sw[T], q, zero);
      static_for<0, 4>([&](auto E) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[E()], q.unit, -sub));
        sum[4 * T + E] += k0 + 16 * T + 4 * c + E < end ? p : 0.0f;
      });
    });
  }
  float mine = 0.0f;  // lane r of a quarter has its slot 16 (r / 4) + 4 c + r % 4
  static_for<0, 16>([&](auto X) {
    float v = sum[X];
    for (int x = 1; x < 16; x *= 2) v += __shfl_xor(v, x);
    mine = r == X ? v : mine;
  });
  sums[wave][16 * (r / 4) + 4 * c + r % 4] = mine;
  __syncthreads();
  if (threadIdx.x >= 64 || k0 + threadIdx.x >= len) return;
  mine = 0.0f;
#pragma unroll
  for (int w = 0; w < NW; w++) mine += sums[w][threadIdx.x];
  a.weight_out[slot + threadIdx.x] = (a.weight ? a.weight[slot + threadIdx.x] : 0.0f) + mine;
}

// What follows the attention kernel: first a workgroup per row whose shares are to be joined, then those of a unit's slots that
// receive weight from stored scores, or of the rows whose operands the slots go by.
template <int NG, int NP>
__global__ void __launch_bounds__(64 * NW) cache4_finish_kernel(Attn4 a, uint32_t joins, uint32_t tile_blocks) {
  const uint32_t x = blockIdx.x - joins;
  if (blockIdx.x < joins) join_row<NG>(a, blockIdx.x);
  else if (a.scores) receive_scores(a, x / tile_blocks, x % tile_blocks);
  else keep_operands<NG, NP>(a, x * NW + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
}
template <int NG, int NP>
__global__ void __launch_bounds__(64 * NW) cache4_receive_kernel(Attn4 a, uint32_t tiles) {
  receive<NG, NP>(a, blockIdx.x / tiles, blockIdx.x % tiles);
}

template <int NG, int NP>
hipError_t launch_np(const Attn4& a, hipStream_t s) {
  const uint32_t units = a.batch * a.kv_heads;
  const dim3 grid((a.split_slots ? a.split_slots : units) * a.row_blocks), block(64 * NW);
  if (grid.x) {
    if (a.pk == 4) hipLaunchKernelGGL((cache4_attention_kernel<NG, 1, NP, 4>), grid, block, 0, s, a);
    else if (a.pk == 2) hipLaunchKernelGGL((cache4_attention_kernel<NG, 1, NP, 2>), grid, block, 0, s, a);
    else if (a.rt == 1) hipLaunchKernelGGL((cache4_attention_kernel<NG, 1, NP, 1>), grid, block, 0, s, a);
    else if constexpr (most_rows(NG) == 2) hipLaunchKernelGGL((cache4_attention_kernel<NG, 2, NP, 1>), grid, block, 0, s, a);
  }
  const uint32_t joins = a.split_slots ? units * a.rows : 0, per = 64 * NW * 4, blocks = (a.max_len + per - 1) / per;
  const uint32_t more = a.scores ? units * blocks : a.operands ? (units * ((a.rows + 15) / 16) + NW - 1) / NW : 0;
  if (joins || more) hipLaunchKernelGGL((cache4_finish_kernel<NG, NP>), dim3(joins + more), block, 0, s, a, joins, blocks);
  if (a.weight_out && !a.scores) {
    const uint32_t tiles = (a.max_len + 63) / 64;
    hipLaunchKernelGGL((cache4_receive_kernel<NG, NP>), dim3(units * tiles), block, 0, s, a, tiles);
  }
  return hipGetLastError();
}

template <int NG>
hipError_t launch_dim(const Attn4& a, hipStream_t s) {
  return a.dtype == F32 ? launch_np<NG, 2>(a, s) : launch_np<NG, 1>(a, s);
}

}  // namespace
}  // namespace we
