// A key / value cache held in 4 bits (include/we_cache4.h): append (quantize), load (dequantize) and eviction by
// accumulated attention weight. Attention over it: cache4_attention.hip.
#include "common.h"
#include "internal.h"

namespace we {
namespace {

__device__ __forceinline__ uint32_t clamped(int32_t v, uint32_t hi) { return v < 0 ? 0u : (uint32_t)v < hi ? (uint32_t)v : hi; }

// ------------------------------------------------------------------------------------------ append
// A thread quantizes 8 consecutive values (one u32 of codes); the 8 lanes of a group of 64 share its range by three lane
// exchanges. Bound by HBM: a row is read once and written once at 4.5 bits a value.
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
    __syncthreads();  // in place, the one workgroup of the sequence has read its length
    if (threadIdx.x == 0) lens_update(a, b, len0, seen0);
  }
}

// ------------------------------------------------------------------------------------------ load
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
// One workgroup per sequence and kv head. The slots to give up are those below the n-th smallest (protected, weight, slot):
// found digit by digit from the top in counts of the slots that share the digits fixed so far; then two passes in slot order
// pair the holes with the survivors that fill them, and the rows move.
struct EvictArgs {
  Cache4Evict a;
};

// f32 as a key of the same order: NaN highest, -0 as 0
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive sum over the 1024 threads' flags in thread order; `total` is the sum of all.
__device__ __forceinline__ uint32_t block_rank(bool flag, uint32_t* waves, uint32_t& total) {
  const uint64_t vote = __ballot(flag);
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
  if (lane == 0) waves[wave] = (uint32_t)__popcll(vote);
  __syncthreads();
  uint32_t before = 0;
  total = 0;
  for (uint32_t w = 0; w < 16; w++) {
    if (w < wave) before += waves[w];
    total += waves[w];
  }
  return before + (uint32_t)__popcll(vote & ((1ull << lane) - 1));
}

__global__ void __launch_bounds__(1024) cache4_evict_kernel(EvictArgs g, uint32_t* from) {
  const Cache4Evict& a = g.a;
  __shared__ uint32_t hist[256], waves[16], found[2];
  const uint32_t gh = blockIdx.x, b = blockIdx.y, t = threadIdx.x, cap = a.c.capacity;
  const uint32_t len = clamped(a.lens[b], a.max_len), left = len < a.keep ? len : a.keep;
  const int64_t young = (int64_t)a.seen[b] - a.recent;
  const size_t base = ((size_t)b * a.c.kv_heads + gh) * cap;
  from += ((size_t)b * a.c.kv_heads + gh) * a.max_len;
  auto prot = [&](uint32_t s) { const int32_t p = a.pos[base + s]; return p < (int32_t)a.sinks || p >= young; };
  // the class the border falls into, and how many of it go
  uint32_t open = 0;
  for (uint32_t s0 = 0; s0 < len; s0 += 1024) {
    uint32_t n;
    block_rank(s0 + t < len && !prot(s0 + t), waves, n);
    open += n;
  }
  uint32_t go = len - left;
  const bool cls = go > open;
  if (cls) go -= open;
  uint32_t prefix = 0, mask = 0;
  if (go) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (t < 256) hist[t] = 0;
      __syncthreads();
      for (uint32_t s = t; s < len; s += 1024) {
        const uint32_t k = order_key(a.weight[base + s]);
        if (prot(s) == cls && (k & mask) == prefix) atomicAdd(&hist[k >> shift & 255u], 1u);
      }
      __syncthreads();
      if (t == 0) {
        uint32_t d = 0, n = go;
        while (hist[d] < n) n -= hist[d++];
        found[0] = d, found[1] = n;
      }
      __syncthreads();
      prefix |= found[0] << shift, mask |= 255u << shift, go = found[1];
    }
  }
  // go: how many of the slots with the border's key go, the lowest first
  uint32_t equal = 0, holes = 0, moves = 0;
  for (uint32_t s0 = 0; s0 < len; s0 += 1024) {
    const uint32_t s = s0 + t;
    bool gone = false, tie = false;
    if (s < len) {
      const bool p = prot(s);
      const uint32_t k = order_key(a.weight[base + s]);
      gone = p != cls ? cls : go && k < prefix;
      tie = p == cls && go && k == prefix;
    }
    uint32_t n;
    const uint32_t rank = equal + block_rank(tie, waves, n);
    equal += n;
    gone |= tie && rank < go;
    const bool hole = gone && s < left, move = !gone && s >= left && s < len;
    const uint32_t hr = holes + block_rank(hole, waves, n);
    holes += n;
    const uint32_t mr = moves + block_rank(move, waves, n);
    moves += n;
    // holes come before every move's slot, so a list of holes below and of sources above fits one array
    if (hole) from[hr] = s;
    if (move) from[a.max_len - 1 - mr] = s;
    if (s < left && !hole) {
      a.weight_out[base + s] = a.weight[base + s];
      a.pos_out[base + s] = a.pos[base + s];
    }
  }
  __syncthreads();
  for (uint32_t m = 0; m < moves; m++) {
    const size_t to = base + from[m], at = base + from[a.max_len - 1 - m];
    const uint32_t words = a.c.dim / 8;
    if (t < words) {
      ((uint32_t*)a.c.kc)[to * words + t] = ((uint32_t*)a.c.kc)[at * words + t];
      ((uint32_t*)a.c.vc)[to * words + t] = ((uint32_t*)a.c.vc)[at * words + t];
    }
    if (t < words / 8) {
      a.c.ks[to * (words / 8) + t] = a.c.ks[at * (words / 8) + t];
      a.c.vs[to * (words / 8) + t] = a.c.vs[at * (words / 8) + t];
    }
    if (t == 0) {
      a.weight_out[to] = a.weight[at];
      a.pos_out[to] = a.pos[at];
    }
  }
}

__global__ void __launch_bounds__(256) cache4_left_kernel(Cache4Evict a) {
  const uint32_t b = blockIdx.x * 256 + threadIdx.x;
  if (b >= a.c.batch) return;
  const uint32_t len = clamped(a.lens[b], a.max_len);
  a.lens_out[b] = (int32_t)(len < a.keep ? len : a.keep);
}

uint32_t blocks_for(uint64_t items) {
  const uint64_t n = (items + 255) / 256;
  return (uint32_t)(n < 1 ? 1 : n < 4096 ? n : 4096);
}

}  // namespace

hipError_t cache4_append_launch(const Cache4Append& L, hipStream_t s) {
  const uint64_t items = (uint64_t)L.tokens * L.c.kv_heads * (L.c.dim / 8) * 2;
  if (items > 0xffffffffull - 4096 * 256) return hipErrorInvalidValue;
  const uint32_t grid = items <= 2048 ? 1 : blocks_for(items);
  AppendArgs g{L, (uint32_t)items, grid > 1};
  const dim3 at(grid, L.c.batch);
  if (L.dtype == F32) hipLaunchKernelGGL(cache4_append_kernel<F32>, at, dim3(256), 0, s, g);
  else if (L.dtype == F16) hipLaunchKernelGGL(cache4_append_kernel<F16>, at, dim3(256), 0, s, g);
  else hipLaunchKernelGGL(cache4_append_kernel<BF16>, at, dim3(256), 0, s, g);
  if (g.late_lens) hipLaunchKernelGGL(cache4_lens_kernel, dim3((L.c.batch + 255) / 256), dim3(256), 0, s, L);
  return hipGetLastError();
}

hipError_t cache4_load_launch(const Cache4Load& L, hipStream_t s) {
  const uint64_t items = (uint64_t)L.tokens * L.c.kv_heads * (L.c.dim / 8) * 2;
  if (items > 0xffffffffull - 4096 * 256) return hipErrorInvalidValue;
  if (!items) return hipSuccess;
  const dim3 at(blocks_for(items), L.c.batch);
  if (L.dtype == F32) hipLaunchKernelGGL(cache4_load_kernel<F32>, at, dim3(256), 0, s, L, (uint32_t)items);
  else if (L.dtype == F16) hipLaunchKernelGGL(cache4_load_kernel<F16>, at, dim3(256), 0, s, L, (uint32_t)items);
  else hipLaunchKernelGGL(cache4_load_kernel<BF16>, at, dim3(256), 0, s, L, (uint32_t)items);
  return hipGetLastError();
}

size_t cache4_evict_scratch(const Cache4Evict& L) { return (size_t)L.c.batch * L.c.kv_heads * L.max_len * 4; }

hipError_t cache4_evict_launch(const Cache4Evict& L, hipStream_t s) {
  hipLaunchKernelGGL(cache4_evict_kernel, dim3(L.c.kv_heads, L.c.batch), dim3(1024), 0, s, EvictArgs{L}, (uint32_t*)L.scratch);
  hipLaunchKernelGGL(cache4_left_kernel, dim3((L.c.batch + 255) / 256), dim3(256), 0, s, L);
  return hipGetLastError();
}

}  // namespace we
