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
#include "common.h"
#include "internal.h"

namespace we {
namespace {

constexpr int NW = 4;          // waves of a workgroup
constexpr float kNone = -3e38f;  // the running maximum before the first score

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
  uint32_t row_blocks;  // of RT * 16 rows
  uint32_t chunk, splits;  // tiles of a split
  float* part;          // splits > 1: O [split][unit][rows][dim], unit = sequence and kv head, times 2^-m
  float* ml;            // and (m, l) [split][unit][rows][2]
  float* lse;           // weights: [unit][rows], log2 of a row's sum of 2^score
};

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
  const f16x2 v0 = __builtin_bit_cast(f16x2, (w & 0x000f000fu) | 0x64006400u) + one;
  const f16x2 v1 = __builtin_bit_cast(f16x2, (w & 0x00f000f0u) | 0x64006400u) + sixteen;
  const f16x2 v2 = __builtin_bit_cast(f16x2, (h & 0x000f000fu) | 0x64006400u) + one;
  const f16x2 v3 = __builtin_bit_cast(f16x2, (h & 0x00f000f0u) | 0x64006400u) + sixteen;
  return u32x4{__builtin_bit_cast(uint32_t, v0), __builtin_bit_cast(uint32_t, v1), __builtin_bit_cast(uint32_t, v2), __builtin_bit_cast(uint32_t, v3)};
}
__device__ __forceinline__ float scale_of(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[0]; }
__device__ __forceinline__ float minimum_of(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[1]; }
__device__ __forceinline__ float middle_of(uint32_t w) { return __builtin_fmaf(scale_of(w), 8.0f, minimum_of(w)); }

// One query row of a lane as MFMA operands: for step (G, s) the 8 values of the codes word 2 c + s of group G, in
// codes_operand's order and factor, times 2^e (largest value below 2^14). NP planes of f16: their sum is q.
template <int NG, int NP>
struct QRow {
  u32x4 f[NG][2][NP];
  float sum[NG];  // of 2^e q over the group, times kCode
  float unit;     // 2^-e log2(e) / sqrt(dim) / kCode: a score in log2 units is unit * (scale . dot + minimum . sum)
  static constexpr float kCode = NP == 1 ? 0x1p-24f : 1.0f;  // what a code of key_operand stands for
};

template <int NG, int NP>
__device__ __forceinline__ void load_row(const Attn4& a, bool live, size_t at, int c, QRow<NG, NP>& q) {
  float x[NG][16];
  float big = 0.0f;
#pragma unroll
  for (int g = 0; g < NG; g++) {
    const size_t i = at + g * 64 + c * 16;
#pragma unroll
    for (int e = 0; e < 16; e++) x[g][e] = 0.0f;
    if (live) {
      if constexpr (NP == 2) {
#pragma unroll
        for (int v = 0; v < 4; v++) {
          const f32x4 w = ((const f32x4*)((const float*)a.q + i))[v];
#pragma unroll
          for (int e = 0; e < 4; e++) x[g][4 * v + e] = w[e];
        }
      } else {
#pragma unroll
        for (int v = 0; v < 2; v++) {
          const u32x4 w = ((const u32x4*)((const uint16_t*)a.q + i))[v];
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const uint16_t h = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
            x[g][8 * v + e] = a.dtype == F16 ? f16_to_f32(h) : bf16_to_f32(h);
          }
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const float v = fabsf(x[g][e]);
      big = fmaxf(big, v < INFINITY ? v : 0.0f);  // an infinite or NaN value stays one in f16, in its own row
    }
  }
  big = row_max(big);
  // 2^e with big 2^e in [2^13, 2^14); e in -98 .. 126, so that `unit` and 2^e are normal numbers
  int e = 13 + 127 - (int)(__float_as_uint(big) >> 23);
  e = e < -98 ? -98 : e > 126 ? 126 : e;
  const float up = __uint_as_float((uint32_t)(e + 127) << 23);
  q.unit = __uint_as_float((uint32_t)(127 - e) << 23) * (1.0f / QRow<NG, NP>::kCode) * a.scale_log2;
#pragma unroll
  for (int g = 0; g < NG; g++) {
    float sum = 0.0f;
#pragma unroll
    for (int s = 0; s < 2; s++) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int lo = s * 8 + j;  // operand register j: codes j and j + 4, the odd j 16 times too large
        const float f = j & 1 ? 0.0625f : 1.0f, p = x[g][lo] * up, r = x[g][lo + 4] * up;
        sum += p + r;
        const uint32_t hi = pack2(p * f, r * f, std::true_type{});
        q.f[g][s][0][j] = hi;
        if constexpr (NP == 2) {
          const f16x2 h = __builtin_bit_cast(f16x2, hi);
          q.f[g][s][1][j] = pack2(p * f - (float)h[0], r * f - (float)h[1], std::true_type{});
        }
      }
    }
    q.sum[g] = row_sum(sum) * QRow<NG, NP>::kCode;
  }
}

// K's operand: the codes as they are, or centred for f32 q, whose scores are worth the four adds.
template <int NP>
__device__ __forceinline__ u32x4 key_operand(uint32_t w) {
  return NP == 1 ? codes_operand(w) : centred_operand(w);
}

// The scores of 16 slots (their codes kf[G], their scale words sw[i * NG + G] for slot i of the lane's four) and a query row,
// before `unit`.
template <int NG, int NP>
__device__ __forceinline__ f32x4 scores(const u32x4 (&kf)[NG][2], const uint32_t (&sw)[4 * NG], const QRow<NG, NP>& q) {
  f32x4 s;
#pragma unroll
  for (int g = 0; g < NG; g++) {
    f32x4 d = {};
#pragma unroll
    for (int p = 0; p < NP; p++) {
      d = mfma_16x16x32<true>(kf[g][0], q.f[g][0][p], d);
      d = mfma_16x16x32<true>(kf[g][1], q.f[g][1][p], d);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float at0 = NP == 1 ? minimum_of(sw[i * NG + g]) : middle_of(sw[i * NG + g]);
      const float m = g == 0 ? at0 * q.sum[0] : __builtin_fmaf(at0, q.sum[g], s[i]);
      s[i] = __builtin_fmaf(scale_of(sw[i * NG + g]), d[i], m);
    }
  }
  return s;
}

__device__ __forceinline__ void unit_of(const Attn4& a, uint32_t unit, uint32_t& len, uint32_t& count) {
  const uint32_t b = unit / a.kv_heads;
  len = in_range(a.lens[b], a.max_len);
  count = a.counts ? in_range(a.counts[b], a.tokens) : a.tokens;
}
// the slots that token i sees
__device__ __forceinline__ uint32_t sees(const Attn4& a, uint32_t len, uint32_t count, uint32_t i) {
  const int32_t n = a.causal ? (int32_t)(len + i + 1) - (int32_t)count : (int32_t)len;
  return n < 0 ? 0u : (uint32_t)n;
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// A stage of a wave's ring: 64 slots as K codes [T][G][16 slots][32 bytes] (so a score step's reads are contiguous), V codes
// [T][16-byte piece][16 slots] (what the transposing read wants), K and V scale words in slot order.
template <int NG>
struct Ring {
  static constexpr int kCodes = 2048 * NG, kScales = 256 * NG, kBytes = 2 * (kCodes + kScales), kStages = 2;
  static constexpr int kLoads = 4 * NG + 2;
};

template <int NG, int RT, int NP>
__global__ void __launch_bounds__(64 * NW, 1) cache4_attention_kernel(Attn4 a) {
  using R = Ring<NG>;
  constexpr int DIM = 64 * NG, ROW = DIM + 4;  // floats of a joined row in LDS, padded against bank conflicts
  static_assert(NW * 16 * ROW * 4 + NW * 16 * 8 <= NW * R::kStages * R::kBytes, "the join fits the ring");
  __shared__ __attribute__((aligned(1024))) char lds[NW * R::kStages * R::kBytes];
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // (unit, split, row block): each XCD takes a run of blocks of one unit, so that the row blocks that read its slots share an
  // L2; the last row blocks first, which see the most
  uint32_t id = blockIdx.x;
  if ((gridDim.x & 7u) == 0u) id = (id & 7u) * (gridDim.x >> 3) + (id >> 3);
  const uint32_t rb = a.row_blocks - 1 - id % a.row_blocks, us = id / a.row_blocks, split = us % a.splits, unit = us / a.splits;
  uint32_t len, count;
  unit_of(a, unit, len, count);
  const uint32_t b = unit / a.kv_heads, gh = unit % a.kv_heads;
  const uint32_t row0 = rb * (RT * 16), rows = count * a.group;
  if (row0 >= rows) return;
  const uint32_t last = row0 + RT * 16 < rows ? row0 + RT * 16 - 1 : rows - 1;
  const uint32_t most = sees(a, len, count, last / a.group), least = sees(a, len, count, row0 / a.group);
  const uint32_t t0 = split * a.chunk;
  uint32_t t1 = (most + 63) / 64;
  t1 = t1 < t0 + a.chunk ? t1 : t0 + a.chunk;

  QRow<NG, NP> q[RT];
  uint32_t vis[RT];
  float m[RT], le[RT], lo[RT], me[RT][NG], mo[RT][NG];  // l and the sum of p (minimum + 8 scale): over even slots i, and odd ones / 16
  f32x4 o[RT][4 * NG];
  static_for<0, RT>([&](auto I) {
    const uint32_t row = row0 + 16 * I + r;
    const bool live = row < rows;
    const uint32_t i = live ? row / a.group : 0, h = live ? row % a.group : 0;
    load_row<NG, NP>(a, live, ((size_t)b * a.tokens + i) * a.q_stride + (size_t)(gh * a.group + h) * DIM, c, q[I]);
    vis[I] = live ? sees(a, len, count, i) : len;
    m[I] = kNone, le[I] = lo[I] = 0.0f;
    static_for<0, NG>([&](auto G) { me[I][G] = mo[I][G] = 0.0f; });
    static_for<0, 4 * NG>([&](auto D) { o[I][D] = f32x4{}; });
  });

  const size_t slots = (size_t)unit * a.capacity;
  const __amdgpu_buffer_rsrc_t rkc = __builtin_amdgcn_make_buffer_rsrc((void*)(a.kc + slots * (32 * NG)), (short)0, (int)(a.capacity * (32 * NG)), 0x00020000);
  const __amdgpu_buffer_rsrc_t rvc = __builtin_amdgcn_make_buffer_rsrc((void*)(a.vc + slots * (32 * NG)), (short)0, (int)(a.capacity * (32 * NG)), 0x00020000);
  const __amdgpu_buffer_rsrc_t rks = __builtin_amdgcn_make_buffer_rsrc((void*)(a.ks + slots * NG), (short)0, (int)(a.capacity * (4 * NG)), 0x00020000);
  const __amdgpu_buffer_rsrc_t rvs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.vs + slots * NG), (short)0, (int)(a.capacity * (4 * NG)), 0x00020000);
  char* ring = lds + wave * (R::kStages * R::kBytes);
  auto issue = [&](uint32_t t, int stage) {
    char* to = ring + stage * R::kBytes;
    static_for<0, 2 * NG>([&](auto J) {
      const uint32_t p = J * 64 + lane;
      const uint32_t tg = p / 32, ko = (16 * (tg / NG) + p % 32 / 2) * (32 * NG) + tg % NG * 32 + p % 2 * 16;
      const uint32_t tc = p / 16, vo = (16 * (tc / (2 * NG)) + p % 16) * (32 * NG) + tc % (2 * NG) * 16;
      dma16s(rkc, to + J * 1024, ko, t * (2048 * NG));
      dma16s(rvc, to + R::kCodes + J * 1024, vo, t * (2048 * NG));
    });
    if (lane < 16 * NG) {
      dma16s(rks, to + 2 * R::kCodes, lane * 16, t * (256 * NG));
      dma16s(rvs, to + 2 * R::kCodes + R::kScales, lane * 16, t * (256 * NG));
    }
  };

  uint32_t slim = 0;   // the largest V scale seen, as f16 bits, rounded up to below a power of two
  float bound = -14.0f;  // log2 of that power
  auto tile = [&](uint32_t t, const char* st, auto MASK) {
    const uint32_t k0 = t * 64 + 4 * c;
    f32x4 s[RT][4];
    static_for<0, 4>([&](auto T) {
      u32x4 kf[NG][2];
      uint32_t sw[4 * NG];
      static_for<0, NG>([&](auto G) {
        const u32x2 w = *(const u32x2*)(st + ((T * NG + G) * 16 + r) * 32 + c * 8);
        kf[G][0] = key_operand<NP>(w.x), kf[G][1] = key_operand<NP>(w.y);
        const u32x4 v = *(const u32x4*)(st + 2 * R::kCodes + (16 * T + 4 * c) * (4 * NG) + G * 16);
        static_for<0, 4>([&](auto E) { sw[4 * G + E] = v[E()]; });
      });
      static_for<0, RT>([&](auto I) { s[I][T] = scores<NG, NP>(kf, sw, q[I]); });
    });
    float mx[RT];
    bool high = false;
    static_for<0, RT>([&](auto I) {
      static_for<0, 4>([&](auto T) {
        static_for<0, 4>([&](auto E) {
          if constexpr (MASK) s[I][T][E()] = k0 + 16 * T + E < vis[I] ? s[I][T][E()] : -INFINITY;
          mx[I] = T + E == 0 ? s[I][0][0] : fmaxf(mx[I], s[I][T][E()]);
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
      static_for<0, 4>([&](auto T) {
        static_for<0, 4>([&](auto E) {
          s[I][T][E()] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[I][T][E()], q[I].unit, -(E & 1 ? odd : even)));
          if constexpr (NP == 2) s[I][T][E()] *= E & 1 ? up * 0.0625f : up;
          if constexpr (E & 1) lo[I] += s[I][T][E()];
          else le[I] += s[I][T][E()];
        });
      });
    });
    uint32_t vw[4][4 * NG];
    static_for<0, 4>([&](auto T) {
      static_for<0, NG>([&](auto G) {
        const u32x4 v = *(const u32x4*)(st + 2 * R::kCodes + R::kScales + (16 * T + 4 * c) * (4 * NG) + G * 16);
        static_for<0, 4>([&](auto E) { vw[T][4 * G + E] = v[E()]; });
      });
    });
    const char* vt = st + R::kCodes + ((r / 4) * (2 * NG * 16) + 4 * c + r % 4) * 16;
    static_for<0, NG>([&](auto G) {
      u32x4 pf[RT][2][NP];
      static_for<0, RT>([&](auto I) {
        static_for<0, 2>([&](auto K) {
          static_for<0, 4>([&](auto E) {
            float p0 = s[I][2 * K][E()], p1 = s[I][2 * K + 1][E()];
            uint32_t w0 = vw[2 * K][E * NG + G], w1 = vw[2 * K + 1][E * NG + G];
            if constexpr (MASK) {  // p is 0 there; the scale may be anything
              w0 = k0 + 32 * K + E < vis[I] ? w0 : 0u;
              w1 = k0 + 32 * K + 16 + E < vis[I] ? w1 : 0u;
            }
            float& mn = E & 1 ? mo[I][G] : me[I][G];
            mn = __builtin_fmaf(p0, middle_of(w0), mn);
            mn = __builtin_fmaf(p1, middle_of(w1), mn);
            p0 *= scale_of(w0), p1 *= scale_of(w1);
            const uint32_t hi = pack2(p0, p1, std::true_type{});
            pf[I][K][0][E()] = hi;
            if constexpr (NP == 2) {
              const f16x2 h = __builtin_bit_cast(f16x2, hi);
              pf[I][K][1][E()] = pack2(p0 - (float)h[0], p1 - (float)h[1], std::true_type{});
            }
          });
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

  uint32_t t = t0 + wave;
  if (t < t1) issue(t, 0);
  if (t + NW < t1) issue(t + NW, 1);
  for (int stage = 0; t < t1; t += NW, stage ^= 1) {
    if (t + NW < t1) wait_loads<R::kLoads>();
    else wait_loads<0>();
    const char* st = ring + stage * R::kBytes;
    if (t * 64 + 64 > least) tile(t, st, std::true_type{});
    else tile(t, st, std::false_type{});
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage's reads are done before it is filled again
    if (t + 2 * NW < t1) issue(t + 2 * NW, stage);
  }

  // join the waves: the largest maximum of a row, every wave's sums brought to it, their total
  float* ml = (float*)lds;                         // [wave][16][2]
  float* joined = ml + NW * 16 * 2;                // [wave][16][ROW]
  static_for<0, RT>([&](auto I) {
    float l = row_sum(le[I] + 16.0f * lo[I]);
    __syncthreads();
    if (c == 0) ml[(wave * 16 + r) * 2] = m[I], ml[(wave * 16 + r) * 2 + 1] = l;
    __syncthreads();
    float top = kNone, total = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; w++) top = fmaxf(top, ml[(w * 16 + r) * 2]);
    const float f = __builtin_amdgcn_exp2f(m[I] - top);
#pragma unroll
    for (int w = 0; w < NW; w++) total += ml[(w * 16 + r) * 2 + 1] * __builtin_amdgcn_exp2f(ml[(w * 16 + r) * 2] - top);
    static_for<0, NG>([&](auto G) {
      const float mn = row_sum(me[I][G] + 16.0f * mo[I][G]);
      static_for<0, 4>([&](auto D) {
        f32x4 v;
        static_for<0, 4>([&](auto E) { v[E()] = f * (o[I][4 * G + D][E()] + mn); });
        *(f32x4*)(joined + (wave * 16 + r) * ROW + (4 * G + D) * 16 + 4 * c) = v;
      });
    });
    __syncthreads();
    if (wave == 0 && c == 0) ml[r * 2] = top, ml[r * 2 + 1] = total;  // read by all below
    __syncthreads();
    for (uint32_t x = threadIdx.x; x < 16 * DIM / 4; x += 64 * NW) {
      const uint32_t rr = x / (DIM / 4), d = x % (DIM / 4) * 4, row = row0 + 16 * I + rr;
      if (row >= rows) continue;
      f32x4 v = {};
#pragma unroll
      for (int w = 0; w < NW; w++) v += *(const f32x4*)(joined + (w * 16 + rr) * ROW + d);
      const float mm = ml[rr * 2], ll = ml[rr * 2 + 1];
      if (a.splits > 1) {
        const size_t at = ((size_t)split * a.batch * a.kv_heads + unit) * a.rows + row;
        *(f32x4*)(a.part + at * DIM + d) = v;
        if (d == 0) a.ml[at * 2] = mm, a.ml[at * 2 + 1] = ll;
        continue;
      }
      if (a.lse && d == 0) a.lse[(size_t)unit * a.rows + row] = mm + __builtin_amdgcn_logf(ll);
      const float inv = ll != 0.0f ? 1.0f / ll : 0.0f;  // 0: a row that sees nothing
      const size_t at = ((size_t)b * a.tokens + row / a.group) * a.out_stride + (size_t)(gh * a.group + row % a.group) * DIM + d;
      if (a.dtype == F32) *(f32x4*)((float*)a.out + at) = v * inv;
      else if (a.dtype == F16) *(u32x2*)((uint16_t*)a.out + at) = u32x2{pack2(v[0] * inv, v[1] * inv, std::true_type{}), pack2(v[2] * inv, v[3] * inv, std::true_type{})};
      else *(u32x2*)((uint16_t*)a.out + at) = u32x2{pack2(v[0] * inv, v[1] * inv, std::false_type{}), pack2(v[2] * inv, v[3] * inv, std::false_type{})};
    }
  });
}

// The splits of a row joined: a thread per four values.
template <int NG>
__global__ void __launch_bounds__(256) cache4_join_kernel(Attn4 a) {
  constexpr int DIM = 64 * NG;
  const uint32_t units = a.batch * a.kv_heads;
  const uint64_t x = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t d = (uint32_t)(x % (DIM / 4)) * 4;
  const uint64_t ur = x / (DIM / 4);
  if (ur >= (uint64_t)units * a.rows) return;
  const uint32_t unit = (uint32_t)(ur / a.rows), row = (uint32_t)(ur % a.rows);
  uint32_t len, count;
  unit_of(a, unit, len, count);
  if (row >= count * a.group) return;
  const uint32_t seen = sees(a, len, count, row / a.group);
  // splits from this on saw nothing of the row's block, or nothing of the row
  const uint32_t splits = min(a.splits, (seen + 64 * a.chunk - 1) / (64 * a.chunk));
  float top = kNone;
  for (uint32_t s = 0; s < splits; s++) top = fmaxf(top, a.ml[((size_t)s * units * a.rows + ur) * 2]);
  float l = 0.0f;
  f32x4 v = {};
  for (uint32_t s = 0; s < splits; s++) {
    const size_t at = (size_t)s * units * a.rows + ur;
    const float f = __builtin_amdgcn_exp2f(a.ml[at * 2] - top);
    l += f * a.ml[at * 2 + 1];
    v += f * *(const f32x4*)(a.part + at * DIM + d);
  }
  if (a.lse && d == 0) a.lse[ur] = top + __builtin_amdgcn_logf(l);
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  const size_t at = ((size_t)(unit / a.kv_heads) * a.tokens + row / a.group) * a.out_stride +
                    (size_t)(unit % a.kv_heads * a.group + row % a.group) * DIM + d;
  if (a.dtype == F32) *(f32x4*)((float*)a.out + at) = v * inv;
  else if (a.dtype == F16) *(u32x2*)((uint16_t*)a.out + at) = u32x2{pack2(v[0] * inv, v[1] * inv, std::true_type{}), pack2(v[2] * inv, v[3] * inv, std::true_type{})};
  else *(u32x2*)((uint16_t*)a.out + at) = u32x2{pack2(v[0] * inv, v[1] * inv, std::false_type{}), pack2(v[2] * inv, v[3] * inv, std::false_type{})};
}

// The attention each slot received: a wave takes 64 slots and walks the query rows, 16 at a time, with their sums known. No
// slot is written by two waves, and the rows are added in one order.
template <int NG, int NP>
__global__ void __launch_bounds__(64 * NW) cache4_weight_kernel(Attn4 a) {
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t unit = blockIdx.y, b = unit / a.kv_heads, gh = unit % a.kv_heads;
  uint32_t len, count;
  unit_of(a, unit, len, count);
  const uint32_t k0 = (blockIdx.x * NW + wave) * 64;
  if (k0 >= len) return;
  const size_t slot = (size_t)unit * a.capacity + k0;
  u32x4 kf[4][NG][2];
  uint32_t sw[4][4 * NG];
  static_for<0, 4>([&](auto T) {
    static_for<0, NG>([&](auto G) {
      const u32x2 w = *(const u32x2*)(a.kc + (slot + 16 * T + r) * (32 * NG) + G * 32 + c * 8);
      kf[T][G][0] = key_operand<NP>(w.x), kf[T][G][1] = key_operand<NP>(w.y);
      const u32x4 v = *(const u32x4*)(a.ks + (slot + 16 * T + 4 * c) * NG + G * 4);
      static_for<0, 4>([&](auto E) { sw[T][4 * G + E] = v[E()]; });
    });
  });
  const uint32_t rows = count * a.group;
  // the first row that sees a slot of the wave's
  const uint32_t first = a.causal && k0 + count > len ? (k0 + count - len) * a.group : 0;
  float sum[16];
  for (int x = 0; x < 16; x++) sum[x] = 0.0f;
  for (uint32_t row0 = first / 16 * 16; row0 < rows; row0 += 16) {
    const uint32_t row = row0 + r;
    const bool live = row < rows;
    const uint32_t i = live ? row / a.group : 0, h = live ? row % a.group : 0;
    QRow<NG, NP> q;
    load_row<NG, NP>(a, live, ((size_t)b * a.tokens + i) * a.q_stride + (size_t)(gh * a.group + h) * (64 * NG), c, q);
    const uint32_t vis = live ? sees(a, len, count, i) : 0;
    const float lse = live ? a.lse[(size_t)unit * a.rows + row] : 0.0f;
    static_for<0, 4>([&](auto T) {
      const f32x4 s = scores<NG, NP>(kf[T], sw[T], q);
      static_for<0, 4>([&](auto E) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[E()], q.unit, -lse));
        sum[4 * T + E] += k0 + 16 * T + 4 * c + E < vis ? p : 0.0f;
      });
    });
  }
  float mine = 0.0f;  // lane r of a quarter writes its slot 16 (r / 4) + 4 c + r % 4
  static_for<0, 16>([&](auto X) {
    float v = sum[X];
    for (int x = 1; x < 16; x *= 2) v += __shfl_xor(v, x);
    mine = r == X ? v : mine;
  });
  const uint32_t k = 16 * (r / 4) + 4 * c + r % 4;
  if (k0 + k < len) a.weight_out[slot + k] = (a.weight ? a.weight[slot + k] : 0.0f) + mine;
}

struct Plan {
  uint32_t rt, row_blocks, chunk, splits;
};

// tiles of 16 query rows that a wave's registers hold
constexpr uint32_t most_rows(int ng) { return ng <= 3 ? 2 : 1; }

Plan plan_of(const Cache4Attention& L) {
  const uint64_t rows = (uint64_t)L.tokens * (L.heads / L.c.kv_heads), units = (uint64_t)L.c.batch * L.c.kv_heads;
  const uint32_t most = most_rows((int)L.c.dim / 64);
  Plan p;
  p.rt = rows <= 16 || most == 1 ? 1 : 2;
  p.row_blocks = (uint32_t)((rows + 16 * p.rt - 1) / (16 * p.rt));
  const uint32_t tiles = (L.max_len + 63) / 64;
  const uint64_t blocks = units * (p.row_blocks ? p.row_blocks : 1);
  // two workgroups a CU; a split of fewer than two tiles a wave costs more to join than it saves
  uint64_t s = (512 + blocks - 1) / blocks;
  const uint64_t top = tiles / (2 * NW);
  s = s < top ? s : top;
  if (s < 1) s = 1;
  p.chunk = (uint32_t)((tiles + s - 1) / s);
  p.splits = p.chunk ? (tiles + p.chunk - 1) / p.chunk : 1;
  return p;
}

template <int NG, int NP>
hipError_t launch(const Attn4& a, const Plan& p, hipStream_t s) {
  const uint32_t units = a.batch * a.kv_heads;
  const dim3 grid(units * p.splits * p.row_blocks), block(64 * NW);
  if (grid.x) {
    if (p.rt == 1) hipLaunchKernelGGL((cache4_attention_kernel<NG, 1, NP>), grid, block, 0, s, a);
    else if constexpr (most_rows(NG) == 2) hipLaunchKernelGGL((cache4_attention_kernel<NG, 2, NP>), grid, block, 0, s, a);
    if (p.splits > 1) {
      const uint64_t threads = (uint64_t)units * a.rows * (16 * NG);
      hipLaunchKernelGGL(cache4_join_kernel<NG>, dim3((uint32_t)((threads + 255) / 256)), dim3(256), 0, s, a);
    }
  }
  if (a.weight_out)
    hipLaunchKernelGGL((cache4_weight_kernel<NG, NP>), dim3((a.max_len + 64 * NW - 1) / (64 * NW), units), block, 0, s, a);
  return hipGetLastError();
}

}  // namespace

size_t cache4_attention_scratch(const Cache4Attention& L) {
  const Plan p = plan_of(L);
  const size_t rows = (size_t)L.c.batch * L.heads * L.tokens;
  return (p.splits > 1 ? p.splits * rows * (L.c.dim + 2) * 4 : 0) + (L.weight_out ? rows * 4 : 0);
}

hipError_t cache4_attention_launch(const Cache4Attention& L, hipStream_t s) {
  const Plan p = plan_of(L);
  const uint64_t units = (uint64_t)L.c.batch * L.c.kv_heads;
  if (units > 65535 || units * p.splits * p.row_blocks > 0x7fffffffull || (uint64_t)L.heads * L.tokens * L.c.batch * (L.c.dim / 4) > 0x7fffffffull * 256)
    return hipErrorInvalidValue;
  Attn4 a{};
  a.kc = L.c.kc, a.ks = L.c.ks, a.vc = L.c.vc, a.vs = L.c.vs, a.q = L.q, a.out = L.out, a.counts = L.counts, a.lens = L.lens;
  a.weight = L.weight, a.weight_out = L.weight_out, a.batch = L.c.batch, a.tokens = L.tokens, a.heads = L.heads;
  a.kv_heads = L.c.kv_heads, a.group = L.heads / L.c.kv_heads, a.capacity = L.c.capacity, a.max_len = L.max_len;
  a.q_stride = L.q_stride, a.out_stride = L.out_stride, a.causal = L.causal, a.dtype = L.dtype;
  a.scale_log2 = 1.4426950408889634f / sqrtf((float)L.c.dim);
  a.rows = L.tokens * a.group, a.row_blocks = p.row_blocks, a.chunk = p.chunk, a.splits = p.splits;
  const size_t rows = (size_t)L.c.batch * L.heads * L.tokens;
  float* at = (float*)L.scratch;
  if (p.splits > 1) a.part = at, a.ml = at + p.splits * rows * L.c.dim, at = a.ml + p.splits * rows * 2;
  if (L.weight_out) a.lse = at;
  const bool two = L.dtype == F32;
  switch (L.c.dim / 64) {
    case 1: return two ? launch<1, 2>(a, p, s) : launch<1, 1>(a, p, s);
    case 2: return two ? launch<2, 2>(a, p, s) : launch<2, 1>(a, p, s);
    case 3: return two ? launch<3, 2>(a, p, s) : launch<3, 1>(a, p, s);
    default: return two ? launch<4, 2>(a, p, s) : launch<4, 1>(a, p, s);
  }
}

}  // namespace we
