// A key / value cache held in 4 bits (include/we_cache4.h): append (quantize), load (dequantize) and eviction by
// accumulated attention weight. Attention over it: cache4_attention.hip.
#include "common.h"
#include "internal.h"

namespace we {
namespace {

__device__ __forceinline__ uint32_t clamped(int32_t v, uint32_t hi) { return v < 0 ? 0u : (uint32_t)v < hi ? (uint32_t)v : hi; }

// ------------------------------------------------------------------------------------------ append
// A thread quantizes 8 consecutive values (one u32 of codes); the 8 lanes of a group of 64 share its range by three lane
// exchanges. Bound by HBM: a row is read once and written once at 4.5 bits a value (6117 tokens of 8 heads of 128, f32: 57 MB
// in 17 us, 3.4 TB/s; one token of 16 sequences 3.4 us, a launch's latency).
struct AppendArgs {
  Cache4Append a;
  uint32_t items;  // 8-value pieces of a sequence: K, then V
  int late_lens;   // the lengths are updated by cache4_lens_kernel
};

template <int DT>
__device__ __forceinline__ void load8(const void* p, size_t i, float (&x)[8]) {
  if constexpr (DT == F32) {
    const f32x4 a = *(const f32x4*)((const float*)p + i), b = *(const f32x4*)((const float*)p + i + 4);
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = a[e], x[4 + e] = b[e];
  } else {
    const u32x4 w = *(const u32x4*)((const uint16_t*)p + i);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const uint16_t h = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
      x[e] = DT == F16 ? f16_to_f32(h) : bf16_to_f32(h);
    }
  }
}
template <int DT>
__device__ __forceinline__ void store8(void* p, size_t i, const float (&x)[8]) {
  if constexpr (DT == F32) {
    *(f32x4*)((float*)p + i) = f32x4{x[0], x[1], x[2], x[3]};
    *(f32x4*)((float*)p + i + 4) = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = pack2(x[2 * e], x[2 * e + 1], std::bool_constant<DT == F16>{});
    *(u32x4*)((uint16_t*)p + i) = w;
  }
}

__device__ __forceinline__ void lens_update(const Cache4Append& a, uint32_t b, int32_t len, int32_t seen) {
  const uint32_t cap = a.c.capacity, n = a.counts ? clamped(a.counts[b], a.tokens) : a.tokens;
  const uint32_t to = clamped(len, cap) + n;
  a.lens_out[b] = (int32_t)(to < cap ? to : cap);
  if (a.seen_out) a.seen_out[b] = seen + (int32_t)n;
}

__global__ void __launch_bounds__(256) cache4_lens_kernel(Cache4Append a) {
  const uint32_t b = blockIdx.x * 256 + threadIdx.x;
  if (b < a.c.batch) lens_update(a, b, a.lens[b], a.seen ? a.seen[b] : a.lens[b]);
}

template <int DT>
__global__ void __launch_bounds__(256) cache4_append_kernel(AppendArgs g) {
  const Cache4Append& a = g.a;
  const uint32_t b = blockIdx.y, cap = a.c.capacity, dim = a.c.dim, words = dim / 8;
  const int32_t len0 = a.lens[b], seen0 = a.seen ? a.seen[b] : len0;
  const uint32_t len = clamped(len0, cap), room = cap - len;
  uint32_t n = a.counts ? clamped(a.counts[b], a.tokens) : a.tokens;
  n = n < room ? n : room;
  // all 8 lanes of a group take the same way: a group's pieces are consecutive items, and 8 divides every count here
  for (uint32_t it = blockIdx.x * 256 + threadIdx.x; it < g.items; it += gridDim.x * 256) {
    const uint32_t w = it % words, row = it / words, rows = g.items / words / 2;
    const bool is_v = row >= rows;
    const uint32_t r = is_v ? row - rows : row, i = r / a.c.kv_heads, h = r % a.c.kv_heads;
    if (i >= n) continue;
    float x[8];
    load8<DT>(is_v ? a.v : a.k, ((size_t)b * a.tokens + i) * (is_v ? a.v_stride : a.k_stride) + (size_t)h * dim + w * 8, x);
    float lo = INFINITY, hi = -INFINITY;
    int nan = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      nan |= x[e] != x[e];
      x[e] = fminf(fmaxf(x[e], -65504.0f), 65504.0f);
      lo = fminf(lo, x[e]), hi = fmaxf(hi, x[e]);
    }
#pragma unroll
    for (int m = 1; m < 8; m *= 2) {
      lo = fminf(lo, __shfl_xor(lo, m)), hi = fmaxf(hi, __shfl_xor(hi, m));
      nan |= __shfl_xor(nan, m);
    }
    uint16_t mn = f32_to_f16(lo), sc = f32_to_f16((hi - lo) / 15.0f);
    if (nan) mn = sc = 0x7e00;
    const float m = f16_to_f32(mn), s = f16_to_f32(sc);
    uint32_t codes = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float u = s > 0.0f ? fminf(fmaxf(rintf((x[e] - m) / s), 0.0f), 15.0f) : 0.0f;
      codes |= (uint32_t)u << (4 * e);
    }
    const uint32_t at = len + i;
    const size_t slot = ((size_t)b * a.c.kv_heads + h) * cap + at;
    ((uint32_t*)(is_v ? a.c.vc : a.c.kc))[slot * words + w] = codes;
    if (w % 8 == 0) (is_v ? a.c.vs : a.c.ks)[slot * (words / 8) + w / 8] = (uint32_t)sc | (uint32_t)mn << 16;
    if (!is_v && w == 0) {
      if (a.pos) a.pos[slot] = seen0 + (int32_t)i;
      if (a.weight) a.weight[slot] = 0.0f;
    }
  }
  if (!g.late_lens && blockIdx.x == 0) {
    __syncthreads();  // in place, this is the sequence's only workgroup and has read its length
    if (threadIdx.x == 0) lens_update(a, b, len0, seen0);
  }
}

// ------------------------------------------------------------------------------------------ load
// The reverse, a thread per 8 values; bound by HBM (57 MB in 14 us, 4.1 TB/s).
template <int DT>
__global__ void __launch_bounds__(256) cache4_load_kernel(Cache4Load a, uint32_t items) {
  const uint32_t b = blockIdx.y, cap = a.c.capacity, dim = a.c.dim, words = dim / 8;
  const uint32_t len = clamped(a.lens[b], cap), first = a.first ? clamped(a.first[b], cap) : 0;
  for (uint32_t it = blockIdx.x * 256 + threadIdx.x; it < items; it += gridDim.x * 256) {
    const uint32_t w = it % words, row = it / words, rows = items / words / 2;
    const bool is_v = row >= rows;
    const uint32_t r = is_v ? row - rows : row, i = r / a.c.kv_heads, h = r % a.c.kv_heads, at = first + i;
    void* to = is_v ? a.v : a.k;
    if (at >= len || !to) continue;
    const size_t slot = ((size_t)b * a.c.kv_heads + h) * cap + at;
    const uint32_t codes = ((const uint32_t*)(is_v ? a.c.vc : a.c.kc))[slot * words + w];
    const uint32_t sm = (is_v ? a.c.vs : a.c.ks)[slot * (words / 8) + w / 8];
    const float s = f16_to_f32((uint16_t)sm), m = f16_to_f32((uint16_t)(sm >> 16));
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = __builtin_fmaf((float)(codes >> (4 * e) & 15u), s, m);  // code * scale is exact in f32
    store8<DT>(to, ((size_t)b * a.tokens + i) * (is_v ? a.v_stride : a.k_stride) + (size_t)h * dim + w * 8, x);
  }
}

// ------------------------------------------------------------------------------------------ evict
// cache4_select_kernel: one workgroup per sequence and kv head finds which slots go and pairs the holes with the survivors
// that fill them; the rows move there too when they are few, else in cache4_move_kernel over the whole chip. A slot's key is
// (protected, weight as an ordered u32): 33 bits, of which the n-th smallest is found in three passes of 12, 11 and 10 bits
// (counts of the slots that share the bits fixed so far). Reads 8 bytes a slot; bound by the latency of those passes. Up to
// 32768 slots a wave holds its keys in registers and the passes run out of LDS; more are read again by each pass. A few
// slots (a decode step of a full cache gives up one) are found one after the other instead. 16 x 4 kv heads, 4097 -> 4096
// slots: 7.2 us (15 by the three passes). 4 x 8, up to 32749 -> 8192: 38 us, of which the loads 3, the passes 14, the lists 16.
constexpr int EV_NT = 1024, EV_WAVES = EV_NT / 64;
constexpr uint32_t EV_ONE_BY_ONE = 4;  // slots to give up that are found one after the other
constexpr uint32_t EV_FEW = 64;  // moves that the selecting workgroup does itself: one step of its 16-lane groups

// f32 as a key of the same order: NaN highest, -0 as 0
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One row from slot `at` to slot `to` (with the base of the unit), by the lanes j = 0 .. 4 NG + 3 of a group.
template <int NG>
__device__ __forceinline__ void move_row(const Cache4Evict& a, size_t to, size_t at, int j) {
  if (j < 4 * NG) {
    uint8_t* p = j < 2 * NG ? a.c.kc : a.c.vc;
    const int o = (j < 2 * NG ? j : j - 2 * NG) * 16;
    *(u32x4*)(p + to * (32 * NG) + o) = *(const u32x4*)(p + at * (32 * NG) + o);
  } else if (j < 4 * NG + 2) {
    uint32_t* p = j == 4 * NG ? a.c.ks : a.c.vs;
#pragma unroll
    for (int x = 0; x < NG; x++) p[to * NG + x] = p[at * NG + x];
  } else if (j == 4 * NG + 2) {
    a.weight_out[to] = a.weight[at];
  } else if (j == 4 * NG + 3) {
    a.pos_out[to] = a.pos[at];
  }
}
template <int NG>
constexpr int kMoveLanes = NG <= 3 ? 16 : 32;

struct EvictArgs {
  Cache4Evict a;
  uint32_t most;     // moves of a unit at most
  uint32_t* counts;  // more than EV_FEW: moves of a unit, and per unit its holes, then the slots that fill them
  uint32_t* lists;
  int late_lens;     // cache4_left_kernel writes lens_out
};

template <int NG, int VPT>
__global__ void __launch_bounds__(EV_NT) cache4_select_kernel(EvictArgs g) {
  const Cache4Evict& a = g.a;
  __shared__ uint32_t hist[4096], waves[2][EV_WAVES], found[3], few[2][EV_FEW];
  __shared__ uint64_t lowest[EV_WAVES];
  const uint32_t gh = blockIdx.x, b = blockIdx.y, unit = b * a.c.kv_heads + gh, cap = a.c.capacity;
  const uint32_t t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t len = clamped(a.lens[b], a.max_len), left = len < a.keep ? len : a.keep;
  const int64_t young = (int64_t)a.seen[b] - a.recent;
  const size_t base = (size_t)unit * cap;
  const float* weight = a.weight + base;
  const int32_t* pos = a.pos + base;
  if (!g.late_lens && gh == 0 && t == 0) a.lens_out[b] = (int32_t)left;
  // out of place, all that is below `left` is copied; the holes there are filled later, by the moves
  if (a.weight_out != a.weight)
    for (uint32_t s = t; s < left; s += EV_NT) a.weight_out[base + s] = weight[s];
  if (a.pos_out != a.pos)
    for (uint32_t s = t; s < left; s += EV_NT) a.pos_out[base + s] = pos[s];
  if (left == len) {
    if (g.most > EV_FEW && t == 0) g.counts[unit] = 0;
    return;
  }

  // the wave's pieces of 64 slots: v = 0 .. pieces - 1 from slot `from` on
  const uint32_t pieces = ((len + 63) / 64 + EV_WAVES - 1) / EV_WAVES, from = wave * pieces * 64;
  uint32_t key[VPT ? VPT : 1], safe[VPT ? (VPT + 31) / 32 : 1] = {};
  auto safe_of = [&](int32_t p) { return p < (int32_t)a.sinks || p >= young; };
  // f(v, in, key, protected) for the wave's pieces
  auto each = [&](auto&& f) {
    if constexpr (VPT > 0) {
#pragma unroll
      for (int v = 0; v < VPT; v++)
        if ((uint32_t)v < pieces) f((uint32_t)v, from + v * 64 + lane < len, key[v], (safe[v / 32] >> (v % 32) & 1u) != 0);
    } else {
      for (uint32_t v = 0; v < pieces; v++) {
        const uint32_t s = from + v * 64 + lane, at = s < len ? s : len - 1;
        f(v, s < len, order_key(weight[at]), safe_of(pos[at]));
      }
    }
  };
  if constexpr (VPT > 0) {
    // eight pieces at a time, so that their loads go out together
#pragma unroll
    for (int v0 = 0; v0 < VPT; v0 += 8) {
      if ((uint32_t)v0 < pieces) {
        float w[8];
        int32_t p[8];
#pragma unroll
        for (int v = 0; v < 8; v++) {
          const uint32_t s = from + (v0 + v) * 64 + lane, at = s < len ? s : len - 1;
          w[v] = weight[at], p[v] = pos[at];
        }
#pragma unroll
        for (int v = 0; v < 8; v++) {
          key[v0 + v] = order_key(w[v]);
          safe[v0 / 32] |= (uint32_t)safe_of(p[v]) << (v0 % 32 + v);
        }
      } else {
#pragma unroll
        for (int v = 0; v < 8; v++) key[v0 + v] = 0;
      }
    }
  }

  uint32_t go = len - left, moves = 0;
  if (go <= EV_ONE_BY_ONE) {
    // one slot or a few (a decode step of a full cache): the lowest, then the lowest above it, ...
    uint64_t last = 0;
    uint32_t gone[EV_ONE_BY_ONE];
#pragma unroll
    for (uint32_t n = 0; n < EV_ONE_BY_ONE; n++) {
      gone[n] = ~0u;
      if (n >= go) continue;
      uint64_t best = ~0ull;
      each([&](uint32_t v, bool in, uint32_t k, bool p) {
        const uint64_t x = ((uint64_t)p << 56 | (uint64_t)k << 24 | (from + v * 64 + lane)) + 1;  // above 0, the first `last`
        if (in && x > last && x < best) best = x;
      });
#pragma unroll
      for (int x = 1; x < 64; x *= 2) {
        const uint64_t y = __shfl_xor(best, x);
        best = y < best ? y : best;
      }
      __syncthreads();
      if (lane == 0) lowest[wave] = best;
      __syncthreads();
      best = lowest[lane % EV_WAVES];
#pragma unroll
      for (int x = 1; x < EV_WAVES; x *= 2) {
        const uint64_t y = __shfl_xor(best, x);
        best = y < best ? y : best;
      }
      last = best;
      gone[n] = (uint32_t)(best - 1) & 0xffffffu;
    }
    auto is_gone = [&](uint32_t s) {
      bool x = false;
#pragma unroll
      for (uint32_t n = 0; n < EV_ONE_BY_ONE; n++) x |= gone[n] == s;
      return x;
    };
    // the holes in order meet the slots from `left` on that stay
    uint32_t fill = left, hole = 0;
    for (uint32_t n = 0; n < go; n++) {
      uint32_t next = ~0u;  // the lowest hole not yet filled
#pragma unroll
      for (uint32_t m = 0; m < EV_ONE_BY_ONE; m++) next = gone[m] < left && gone[m] >= hole && gone[m] < next ? gone[m] : next;
      if (next == ~0u) break;
      while (is_gone(fill)) fill++;
      if (g.most <= EV_FEW) {
        if (t / kMoveLanes<NG> == n) move_row<NG>(a, base + next, base + fill, (int)(t % kMoveLanes<NG>));
      } else if (t == 0) {
        uint32_t* list = g.lists + (size_t)unit * 2 * g.most;
        list[n] = next, list[g.most + n] = fill;
      }
      hole = next + 1, fill++, moves++;
    }
    if (g.most > EV_FEW && t == 0) g.counts[unit] = moves;
    return;
  }

  // the border: its class and key, and how many of the slots that have them go
  uint32_t prefix = 0;
  bool cls = false;
  auto narrow = [&](auto BITS, int shift, uint32_t mask) {
    constexpr uint32_t bins = 1u << BITS;
    __syncthreads();
    for (uint32_t x = t; x < bins; x += EV_NT) hist[x] = 0;
    __syncthreads();
    each([&](uint32_t, bool in, uint32_t k, bool p) {
      const uint32_t d = mask ? k >> shift & (bins - 1) : k >> shift | (uint32_t)p << 11;
      if (in && (mask == 0 || (p == cls && (k & mask) == prefix))) atomicAdd(&hist[d], 1u);
    });
    __syncthreads();
    // which bin the go-th falls into: each thread sums its bins, waves by lane exchange
    constexpr uint32_t own = bins < EV_NT ? 1 : bins / EV_NT;
    uint32_t c[own], sum = 0;
#pragma unroll
    for (uint32_t x = 0; x < own; x++) {
      c[x] = t * own + x < bins ? hist[t * own + x] : 0;
      sum += c[x];
    }
    uint32_t up = sum;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
      const uint32_t n = (uint32_t)__shfl_up((int)up, x);
      up += lane >= (uint32_t)x ? n : 0;
    }
    if (lane == 63) waves[0][wave] = up;
    __syncthreads();
    uint32_t before = up - sum;
#pragma unroll
    for (uint32_t w = 0; w < EV_WAVES; w++) before += w < wave ? waves[0][w] : 0;
#pragma unroll
    for (uint32_t x = 0; x < own; x++) {
      if (before < go && go <= before + c[x]) found[0] = t * own + x, found[1] = go - before, found[2] = c[x];
      before += c[x];
    }
    __syncthreads();
    go = found[1];
    return found[0];
  };
  uint32_t d = narrow(std::integral_constant<int, 12>{}, 21, 0u);
  cls = d >> 11;
  prefix = d << 21;
  d = narrow(std::integral_constant<int, 11>{}, 10, 0xffe00000u);
  prefix |= d << 10;
  d = narrow(std::integral_constant<int, 10>{}, 0, 0xfffffc00u);
  prefix |= d;

  // In slot order, so that holes and survivors are numbered: a wave's slots are consecutive, and the waves before it have
  // counted theirs. Where not all slots with the border's key go, the lowest do: those are numbered first.
  const bool all_ties = found[2] == go;
  uint32_t ties = 0;
  if (!all_ties) {
    each([&](uint32_t, bool in, uint32_t k, bool p) { ties += (uint32_t)__popcll(__ballot(in && p == cls && k == prefix)); });
    __syncthreads();
    if (lane == 0) waves[0][wave] = ties;
    __syncthreads();
    ties = 0;
    for (uint32_t w = 0; w < wave; w++) ties += waves[0][w];
  }
  const uint32_t first_tie = ties;
  const uint64_t below = (1ull << lane) - 1;
  auto gone_of = [&](bool in, uint32_t k, bool p) {
    bool tie = k == prefix;
    if (!all_ties) {
      const uint64_t who = __ballot(in && p == cls && tie);
      tie = tie && ties + (uint32_t)__popcll(who & below) < go;
      ties += (uint32_t)__popcll(who);
    }
    return in && (p != cls ? cls : k < prefix || tie);
  };
  uint32_t holes = 0, fills = 0;
  each([&](uint32_t v, bool in, uint32_t k, bool p) {
    const uint32_t s0 = from + v * 64;  // a piece lies below `left`, above it, or across
    const bool gone = gone_of(in, k, p);
    if (s0 < left) holes += (uint32_t)__popcll(__ballot(gone && s0 + lane < left));
    if (s0 + 64 > left) fills += (uint32_t)__popcll(__ballot(in && !gone && s0 + lane >= left));
  });
  __syncthreads();
  if (lane == 0) waves[0][wave] = holes, waves[1][wave] = fills;
  __syncthreads();
  holes = fills = 0;
  for (uint32_t w = 0; w < EV_WAVES; w++) {
    if (w < wave) holes += waves[0][w], fills += waves[1][w];
    moves += waves[0][w];
  }
  uint32_t* hole_list = g.most <= EV_FEW ? few[0] : g.lists + (size_t)unit * 2 * g.most;
  uint32_t* fill_list = g.most <= EV_FEW ? few[1] : hole_list + g.most;
  ties = first_tie;
  each([&](uint32_t v, bool in, uint32_t k, bool p) {
    const uint32_t s0 = from + v * 64, s = s0 + lane;
    const bool gone = gone_of(in, k, p);
    if (s0 < left) {
      const bool hole = gone && s < left;
      const uint64_t h = __ballot(hole);
      if (hole) hole_list[holes + (uint32_t)__popcll(h & below)] = s;
      holes += (uint32_t)__popcll(h);
    }
    if (s0 + 64 > left) {
      const bool fill = in && !gone && s >= left;
      const uint64_t f = __ballot(fill);
      if (fill) fill_list[fills + (uint32_t)__popcll(f & below)] = s;
      fills += (uint32_t)__popcll(f);
    }
  });
  if (g.most <= EV_FEW) {
    __syncthreads();
    constexpr int L = kMoveLanes<NG>;
    for (uint32_t m = t / L; m < moves; m += EV_NT / L) move_row<NG>(a, base + few[0][m], base + few[1][m], (int)(t % L));
  } else if (t == 0) {
    g.counts[unit] = moves;
  }
}

// Bound by HBM: a row is read and written once, 16 bytes a lane (4 x 8 kv heads, up to 32749 -> 8192 slots: 18 us, 3 TB/s).
template <int NG>
__global__ void __launch_bounds__(256) cache4_move_kernel(EvictArgs g) {
  constexpr uint32_t L = kMoveLanes<NG>;
  const uint32_t unit = blockIdx.y, moves = g.counts[unit];
  const uint32_t* holes = g.lists + (size_t)unit * 2 * g.most;
  const size_t base = (size_t)unit * g.a.c.capacity;
  for (uint32_t m = (blockIdx.x * 256 + threadIdx.x) / L; m < moves; m += gridDim.x * (256 / L))
    move_row<NG>(g.a, base + holes[m], base + holes[g.most + m], (int)(threadIdx.x % L));
}

__global__ void __launch_bounds__(256) cache4_left_kernel(Cache4Evict a) {
  const uint32_t b = blockIdx.x * 256 + threadIdx.x;
  if (b >= a.c.batch) return;
  const uint32_t len = clamped(a.lens[b], a.max_len);
  a.lens_out[b] = (int32_t)(len < a.keep ? len : a.keep);
}

template <int NG>
void launch_evict(const EvictArgs& g, hipStream_t s) {
  const Cache4Evict& a = g.a;
  const dim3 units(a.c.kv_heads, a.c.batch);
  if (a.max_len <= 8 * EV_NT) hipLaunchKernelGGL((cache4_select_kernel<NG, 8>), units, dim3(EV_NT), 0, s, g);
  else if (a.max_len <= 32 * EV_NT) hipLaunchKernelGGL((cache4_select_kernel<NG, 32>), units, dim3(EV_NT), 0, s, g);
  else hipLaunchKernelGGL((cache4_select_kernel<NG, 0>), units, dim3(EV_NT), 0, s, g);
  if (g.most > EV_FEW) {
    const uint32_t n = a.c.kv_heads * a.c.batch, per = 256 / kMoveLanes<NG>;
    uint32_t blocks = (g.most + per - 1) / per;
    const uint32_t fill = 4096 / n + 1;  // 16 workgroups a CU in all
    hipLaunchKernelGGL(cache4_move_kernel<NG>, dim3(blocks < fill ? blocks : fill, n), dim3(256), 0, s, g);
  }
}

uint32_t blocks_for(uint64_t items) {
  const uint64_t n = (items + 255) / 256;
  return (uint32_t)(n < 1 ? 1 : n < 4096 ? n : 4096);
}

}  // namespace

hipError_t cache4_append_launch(const Cache4Append& L, hipStream_t s) {
  const uint64_t items = (uint64_t)L.tokens * L.c.kv_heads * (L.c.dim / 8) * 2;
  const uint32_t grid = items <= 2048 ? 1 : blocks_for(items);
  // in place, the lengths change when every workgroup of their sequence has read them
  AppendArgs g{L, (uint32_t)items, grid > 1 && (L.lens_out == L.lens || L.seen_out == L.seen)};
  const dim3 at(grid, L.c.batch);
  if (L.dtype == F32) hipLaunchKernelGGL(cache4_append_kernel<F32>, at, dim3(256), 0, s, g);
  else if (L.dtype == F16) hipLaunchKernelGGL(cache4_append_kernel<F16>, at, dim3(256), 0, s, g);
  else hipLaunchKernelGGL(cache4_append_kernel<BF16>, at, dim3(256), 0, s, g);
  if (g.late_lens) hipLaunchKernelGGL(cache4_lens_kernel, dim3((L.c.batch + 255) / 256), dim3(256), 0, s, L);
  return hipGetLastError();
}

hipError_t cache4_load_launch(const Cache4Load& L, hipStream_t s) {
  const uint64_t items = (uint64_t)L.tokens * L.c.kv_heads * (L.c.dim / 8) * 2;
  if (!items) return hipSuccess;
  const dim3 at(blocks_for(items), L.c.batch);
  if (L.dtype == F32) hipLaunchKernelGGL(cache4_load_kernel<F32>, at, dim3(256), 0, s, L, (uint32_t)items);
  else if (L.dtype == F16) hipLaunchKernelGGL(cache4_load_kernel<F16>, at, dim3(256), 0, s, L, (uint32_t)items);
  else hipLaunchKernelGGL(cache4_load_kernel<BF16>, at, dim3(256), 0, s, L, (uint32_t)items);
  return hipGetLastError();
}

namespace {
uint32_t most_moves(const Cache4Evict& L) {
  const uint32_t out = L.max_len > L.keep ? L.max_len - L.keep : 0;
  return out < L.keep ? out : L.keep;
}
}  // namespace

size_t cache4_evict_scratch(const Cache4Evict& L) {
  const uint32_t most = most_moves(L);
  return most <= EV_FEW ? 0 : (size_t)L.c.batch * L.c.kv_heads * (1 + 2 * (size_t)most) * 4;
}

hipError_t cache4_evict_launch(const Cache4Evict& L, hipStream_t s) {
  if ((uint64_t)L.c.batch * L.c.kv_heads > 65535) return hipErrorInvalidValue;
  EvictArgs g{L, most_moves(L), (uint32_t*)L.scratch, (uint32_t*)L.scratch + (size_t)L.c.batch * L.c.kv_heads, L.lens_out == L.lens};
  switch (L.c.dim / 64) {
    case 1: launch_evict<1>(g, s); break;
    case 2: launch_evict<2>(g, s); break;
    case 3: launch_evict<3>(g, s); break;
    default: launch_evict<4>(g, s); break;
  }
  // in place, the lengths change when every kv head has read them
  if (g.late_lens) hipLaunchKernelGGL(cache4_left_kernel, dim3((L.c.batch + 255) / 256), dim3(256), 0, s, L);
  return hipGetLastError();
}

}  // namespace we
