// The experts of a token, and its rows on their way to them and back.
//
// Choice. p = softmax(z) over the experts' logits; the k largest, equal ones by
// index, with weights scale p (or scale p over their sum). A logit of -inf is never
// chosen: an entry without an expert has id -1, weight 0 and no place.
// Order. The (token, expert) pairs sorted by expert, tokens in order within one:
// offsets[e] is expert e's first place, slots[pair] a pair's place, rows[place] its
// token. Counting sort: each block counts its tokens' pairs an expert, adds what
// the blocks before it counted, and ranks its own. No atomic's order reaches a
// result.
// Rows. spread: y[slots[t, j]] = w[t, j] x[t], and the weights' gradients x[t] .
// y_old; combine: out[t] = resid[t] + sum_j w[t, j] y[slots[t, j]], in order of j.
// Each is the other's backward.
#include <cmath>

#include "mr_rows.h"

namespace mr {
namespace {

// ---- choice -----------------------------------------------------------------

constexpr int kRouteThreads = 1024;
constexpr int kRouteWaves = kRouteThreads / 64;
constexpr int kMaxExperts = 512, kMaxTop = 64;

struct RouteParams {
  const void* z;
  int64_t ldz;
  int T, E, k;
  bool normalize, whole;  // whole: a row is runs of four on addresses of their size
  float scale;
  float* weights;
  int32_t* ids;
  int32_t* offsets;  // null: no order is asked for
  int32_t* slots;
  int32_t* rows;
  int32_t* counts;   // [blocks, E], of several blocks
  int chunk;         // tokens of a block
  int blocks;
};

// A float's place in the descending order as an unsigned number: NaN above all,
// -inf (which is never chosen) at 0, zeros alike. And back: the float (of a NaN, one).
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  if (x == -INFINITY) return 0;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}

// x reduced over the L lanes of a token (L = 16, 32 or 64, aligned).
template <int L, typename T, typename F>
__device__ __forceinline__ T lanes_reduce(T x, F f) {
  x = f(x, dpp<kDppXor1>(x));
  x = f(x, dpp<kDppXor2>(x));
  x = f(x, dpp<kDppHalfMirror>(x));
  x = f(x, dpp<kDppMirror>(x));
  if constexpr (L >= 32) x = f(x, __shfl_xor(x, 16, 64));
  if constexpr (L >= 64) x = f(x, __shfl_xor(x, 32, 64));
  return x;
}

// A token's logits, V to a lane, runs of four: the expert of a lane's entry i.
template <int L>
constexpr __device__ __forceinline__ int expert_of(int i, int l) { return i / 4 * (4 * L) + l * 4 + i % 4; }

template <int DT, int L, int V>
__device__ __forceinline__ void load_logits(const RouteParams& p, int64_t t, int l, float (&z)[V]) {
  const char* row = static_cast<const char*>(p.z) + t * p.ldz * (DT == MR_F32 ? 4 : 2);
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    const int e = expert_of<L>(i, l);
    if (p.whole) {  // (runs lie wholly inside or past the row, on addresses of their size)
      if (e < p.E) {
        if constexpr (DT == MR_F32) {
          const float4 v = *reinterpret_cast<const float4*>(row + e * 4);
          z[i] = v.x, z[i + 1] = v.y, z[i + 2] = v.z, z[i + 3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(row + e * 2);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t w = (k < 2 ? v.x : v.y) >> (16 * (k & 1));
            z[i + k] = DT == MR_BF16 ? __uint_as_float(w << 16) : f16_to_f32(static_cast<uint16_t>(w));
          }
        }
      } else {
        z[i] = z[i + 1] = z[i + 2] = z[i + 3] = -INFINITY;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) z[i + k] = e + k < p.E ? load_elem<DT>(row, e + k) : -INFINITY;
    }
  }
}

// The block's tokens t0 .. t1 - 1: ids and weights, and the count of each expert in
// hist (LDS). A choice is a maximum over the lanes; what is chosen leaves the keys.
// 16-bit logits make one key with their expert (the upper half in order, the lower
// the expert from the top): the maximum is the choice. 32-bit ones need a second
// reduction, over the lanes that hold the maximum, for the lowest expert. The
// instructions of the choices bound it, 30 to 50 each (16384 tokens, 8 of 128 experts:
// 13 us with the order; with the value fetched from its lane and 64 tokens for half the
// CUs 20).
template <int DT, int L, int V>
__device__ __forceinline__ void choose(const RouteParams& p, int t0, int t1, int32_t* hist) {
  constexpr int TOKENS = kRouteThreads / L;
  constexpr bool NARROW = DT != MR_F32;
  const int l = threadIdx.x % L;
  auto largest = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  auto least = [](uint32_t a, uint32_t b) { return a < b ? a : b; };
  for (int t = t0 + static_cast<int>(threadIdx.x) / L; t < t1; t += TOKENS) {
    float z[V];
    load_logits<DT, L, V>(p, t, l, z);
    uint32_t key[V];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      key[i] = order_key(z[i]);
      if constexpr (NARROW) {
        // (a 16-bit float's key: of bf16 the upper half, of fp16, whose values need 13 bits
        // more than the half has, the order of its own bits)
        uint32_t k16 = key[i] >> 16;
        if constexpr (DT == MR_F16) {
          const uint32_t b = f32_to_f16(z[i] + 0.0f);
          k16 = key[i] == 0 ? 0 : key[i] == 0xffffffffu ? 0xffffu : (b & 0x8000u) ? ~b & 0xffffu : b | 0x8000u;
        }
        key[i] = key[i] == 0 ? 0 : (k16 << 16) | (0xffffu - expert_of<L>(i, l));
      }
      m = fmaxf(m, z[i]);
    }
    m = lanes_reduce<L>(m, [](float a, float b) { return fmaxf(a, b); });
    float sum = 0.0f;
    if (!p.normalize && m > -INFINITY) {  // (of NaN and +inf: NaN, like every weight then)
#pragma unroll
      for (int i = 0; i < V; ++i) sum += expf(z[i] - m);
      sum = lanes_reduce<L>(sum, [](float a, float b) { return a + b; });
    }
    float own = -INFINITY;  // the logit of this lane's entry, entry l
    int own_id = -1;
    for (int j = 0; j < p.k; ++j) {
      uint32_t best = key[0];
#pragma unroll
      for (int i = 1; i < V; ++i) best = largest(best, key[i]);
      const uint32_t top = lanes_reduce<L>(best, largest);
      uint32_t at;
      if constexpr (NARROW) {
        at = 0xffffu - (top & 0xffffu);
#pragma unroll
        for (int i = 0; i < V; ++i) key[i] = key[i] == top ? 0 : key[i];
      } else {
        at = 0xffffffffu;
#pragma unroll
        for (int i = V - 1; i >= 0; --i) at = key[i] == top ? expert_of<L>(i, l) : at;
        at = lanes_reduce<L>(at, least);
#pragma unroll
        for (int i = 0; i < V; ++i) key[i] = at == static_cast<uint32_t>(expert_of<L>(i, l)) ? 0 : key[i];
      }
      if (l == j && top) {
        if constexpr (DT == MR_F32) {
          own = key_value(top);
        } else if constexpr (DT == MR_BF16) {
          own = key_value((top & 0xffff0000u) | ((top & 0x80000000u) ? 0 : 0xffffu));
        } else {
          const uint32_t k = top >> 16;
          own = f16_to_f32(static_cast<uint16_t>((k & 0x8000u) ? k ^ 0x8000u : ~k));
        }
        own_id = static_cast<int>(at);
      }
    }
    float w = own_id >= 0 ? expf(own - m) : 0.0f;
    if (p.normalize) sum = lanes_reduce<L>(w, [](float a, float b) { return a + b; });
    w = own_id >= 0 ? w / sum * p.scale : 0.0f;
    if (l < p.k) {
      const int64_t at = static_cast<int64_t>(t) * p.k + l;
      p.ids[at] = own_id;
      p.weights[at] = w;
      if (own_id >= 0 && p.offsets) atomicAdd(hist + own_id, 1);
    }
  }
}

// ---- order ------------------------------------------------------------------

// start[e]: the place of the block's first pair of expert e. hist[e], its own
// count, where it is the only block; else counts[.][e].
__device__ __forceinline__ void block_starts(const RouteParams& p, const int32_t* hist, int32_t* start, int32_t* scratch) {
  const int tid = threadIdx.x, E = p.E;
  int32_t all = 0, before = 0;
  if (p.blocks == 1) {
    if (tid < E) all = hist[tid];
  } else {
    // runs of blocks by groups of threads (E a group), added in LDS
    const int wide = (E + 63) / 64 * 64, groups = kRouteThreads / wide, g = tid / wide, e = tid % wide;
    int32_t a = 0, b = 0;
    if (g < groups && e < E) {
      const int per = (p.blocks + groups - 1) / groups;
      const int32_t* c = p.counts + e;
#pragma unroll 16
      for (int i = g * per; i < min((g + 1) * per, p.blocks); ++i) {
        const int32_t n = c[static_cast<int64_t>(i) * E];
        a += n;
        b += i < static_cast<int>(blockIdx.x) ? n : 0;
      }
    }
    if (tid < E) scratch[tid] = start[tid] = 0;
    __syncthreads();
    if (g < groups && e < E) {
      atomicAdd(scratch + e, a);
      atomicAdd(start + e, b);
    }
    __syncthreads();
    if (tid < E) {
      all = scratch[tid];
      before = start[tid];
    }
    __syncthreads();
  }
  // exclusive scan of the experts' counts over the threads
  const int lane = tid & 63;
  const int32_t upto = wave_scan(all);
  if (lane == 63) scratch[tid >> 6] = upto;
  __syncthreads();
  int32_t base = 0;
  for (int w = 0; w < (tid >> 6); ++w) base += scratch[w];
  const int32_t first = base + upto - all;
  if (tid < E) start[tid] = first + before;
  if (blockIdx.x == 0 && tid < E) {
    p.offsets[tid] = first;
    if (tid == E - 1) p.offsets[E] = first + all;
  }
  __syncthreads();
}

// The places of the block's pairs: its waves take runs of pairs in order. A wave
// counts its run's experts in its row of `of_wave`; the rows become the places
// where each wave's pairs of an expert start; then 64 pairs at a time, the lanes of
// one expert (found bit by bit) take consecutive places.
__device__ __forceinline__ void place(const RouteParams& p, int t0, int t1, const int32_t* start, int32_t* of_wave) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, E = p.E;
  const int64_t first = static_cast<int64_t>(t0) * p.k;
  const int64_t pairs = static_cast<int64_t>(t1 - t0) * p.k;
  const int64_t per = ((pairs + kRouteWaves - 1) / kRouteWaves + 63) / 64 * 64;
  const int64_t a = wave * per, b = min(a + per, pairs);
  int32_t* mine = of_wave + wave * E;
  for (int e = lane; e < E; e += 64) mine[e] = 0;
  __syncthreads();
  int first_id = -1;  // of the run's first 64 pairs, which is all there are of most runs
  for (int64_t i = a + lane; i < b; i += 64) {
    const int id = p.ids[first + i];
    first_id = i < a + 64 ? id : first_id;
    if (id >= 0) atomicAdd(mine + id, 1);
  }
  __syncthreads();
  if (tid < E) {
    int32_t at = start[tid], n[kRouteWaves];
#pragma unroll
    for (int w = 0; w < kRouteWaves; ++w) n[w] = of_wave[w * E + tid];
#pragma unroll
    for (int w = 0; w < kRouteWaves; ++w) {
      of_wave[w * E + tid] = at;
      at += n[w];
    }
  }
  __syncthreads();
  int bits = 0;
  while ((1 << bits) < E) ++bits;
  for (int64_t i = a; i < b; i += 64) {
    const int64_t pair = first + i + lane;
    const int id = i == a ? first_id : i + lane < b ? p.ids[pair] : -1;
    uint64_t same = __ballot(id >= 0);
    for (int q = 0; q < bits; ++q) {
      const uint64_t set = __ballot((id >> q) & 1);
      same &= ((id >> q) & 1) ? set : ~set;
    }
    const int leader = same ? __builtin_ctzll(same) : 0;
    int32_t at = 0;
    if (id >= 0 && lane == leader) at = atomicAdd(mine + id, static_cast<int32_t>(__popcll(same)));
    at = __shfl(at, leader, 64);
    if (i + lane < b) {
      if (id >= 0) {
        at += __popcll(same & ((1ull << lane) - 1));
        p.slots[pair] = at;
        p.rows[at] = static_cast<int32_t>(pair / p.k);
      } else {
        p.slots[pair] = -1;
      }
    }
  }
}

// LDS of a block: counts or starts [E], scratch [E], places a wave [waves, E].
constexpr size_t route_lds(int64_t E) { return static_cast<size_t>(E * (2 + kRouteWaves) + 16) * 4; }

template <int DT, int L, int V>
__global__ __launch_bounds__(kRouteThreads) void route_choose(RouteParams p) {
  extern __shared__ int32_t lds[];
  int32_t* hist = lds;
  for (int e = threadIdx.x; e < p.E; e += kRouteThreads) hist[e] = 0;
  __syncthreads();
  const int t0 = static_cast<int>(blockIdx.x) * p.chunk, t1 = min(t0 + p.chunk, p.T);
  choose<DT, L, V>(p, t0, t1, hist);
  if (!p.offsets) return;
  __syncthreads();  // (the block's ids too)
  if (p.blocks > 1) {
    for (int e = threadIdx.x; e < p.E; e += kRouteThreads) p.counts[static_cast<int64_t>(blockIdx.x) * p.E + e] = hist[e];
    return;
  }
  block_starts(p, hist, lds + p.E, lds + 2 * p.E);
  place(p, t0, t1, lds + p.E, lds + 2 * p.E);
}

__global__ __launch_bounds__(kRouteThreads) void route_place(RouteParams p) {
  extern __shared__ int32_t lds[];
  const int t0 = static_cast<int>(blockIdx.x) * p.chunk, t1 = min(t0 + p.chunk, p.T);
  block_starts(p, lds, lds + p.E, lds + 2 * p.E);
  place(p, t0, t1, lds + p.E, lds + 2 * p.E);
}

// The gradient of the logits: dz = p (d - sum p d), d the weights' gradients at
// the chosen experts; over the chosen alone where their weights were normalized.
struct RouteBwdParams {
  RouteParams f;
  const float* dw;
  void* dz;
  int64_t lddz;
};
// What the chosen experts get goes to their places in LDS and back to the lanes that
// hold them (16384 tokens of 256 experts, 8 chosen: 9.6 us, 3.6 TB/s; with every
// logit's place compared with every chosen one 15).
template <int DT, int L, int V>
__global__ __launch_bounds__(256) void route_bwd(RouteBwdParams p) {
  constexpr int TOKENS = 256 / L, E = L * V;
  __shared__ __attribute__((aligned(16))) float d_of[TOKENS][E];
  __shared__ __attribute__((aligned(16))) uint8_t chosen_of[TOKENS][E];
  const int l = threadIdx.x % L, mine = threadIdx.x / L, k = p.f.k;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * TOKENS + mine;
  const bool there = t < p.f.T;  // (whole groups of L lanes, which reduce among themselves)
  float z[V];
  if (there) load_logits<DT, L, V>(p.f, t, l, z);
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    *reinterpret_cast<float4*>(&d_of[mine][expert_of<L>(i, l)]) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    *reinterpret_cast<uint32_t*>(&chosen_of[mine][expert_of<L>(i, l)]) = 0;
  }
  __syncthreads();
  if (there && l < k) {
    const int id = p.f.ids[t * k + l];
    if (id >= 0 && id < p.f.E) {
      d_of[mine][id] = p.dw[t * k + l];
      chosen_of[mine][id] = 1;
    }
  }
  __syncthreads();
  if (!there) return;
  float d[V];
  bool chosen[V];
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(&d_of[mine][expert_of<L>(i, l)]);
    const uint32_t c = *reinterpret_cast<const uint32_t*>(&chosen_of[mine][expert_of<L>(i, l)]);
    d[i] = v.x, d[i + 1] = v.y, d[i + 2] = v.z, d[i + 3] = v.w;
#pragma unroll
    for (int q = 0; q < 4; ++q) chosen[i + q] = (c >> (8 * q)) & 1;
  }
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (p.f.normalize && !chosen[i]) z[i] = -INFINITY;
    m = fmaxf(m, z[i]);
  }
  m = lanes_reduce<L>(m, [](float a, float b) { return fmaxf(a, b); });
  float e[V], sum = 0.0f, dot = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    e[i] = m > -INFINITY ? expf(z[i] - m) : z[i] == -INFINITY ? 0.0f : z[i];  // (z a NaN: a row of them and -inf)
    sum += e[i];
    dot += e[i] * d[i];
  }
  sum = lanes_reduce<L>(sum, [](float a, float b) { return a + b; });
  dot = lanes_reduce<L>(dot, [](float a, float b) { return a + b; });
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // (a row that is -inf throughout has no gradient)
  dot *= inv;
  char* const row = static_cast<char*>(p.dz) + t * p.lddz * (DT == MR_F32 ? 4 : 2);
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    const int at = expert_of<L>(i, l);
    float g[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) g[q] = p.f.scale * (e[i + q] * inv) * (d[i + q] - dot);
    if (p.f.whole) {
      if (at >= p.f.E) continue;
      if constexpr (DT == MR_F32) {
        *reinterpret_cast<float4*>(row + at * 4) = make_float4(g[0], g[1], g[2], g[3]);
      } else if constexpr (DT == MR_BF16) {
        *reinterpret_cast<uint2*>(row + at * 2) = make_uint2(pack_bf16x2(g[0], g[1]), pack_bf16x2(g[2], g[3]));
      } else {
        *reinterpret_cast<uint2*>(row + at * 2) =
            make_uint2(f32_to_f16(g[0]) | static_cast<uint32_t>(f32_to_f16(g[1])) << 16,
                       f32_to_f16(g[2]) | static_cast<uint32_t>(f32_to_f16(g[3])) << 16);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (at + q < p.f.E) store_elem<DT>(row, at + q, g[q]);
    }
  }
}

// ---- rows -------------------------------------------------------------------

struct RowsParams {
  const void* x;    // spread: [T, H] rows; combine: resid or null
  int64_t ldx;
  void* y;          // the experts' rows [R, H] (spread writes, combine reads)
  int64_t ldy;
  const void* y_old;  // spread: what the weights' gradients multiply, or null
  int64_t ldyo;
  int64_t R;
  const int32_t* slots;
  const float* weights;  // [T, k] or null
  float* dweights;       // spread: [T, k] or null
  void* out;
  int64_t ldo;
  int64_t T;
  int H, k, pieces;
};

// Eight places at a time are in flight; a place outside the rows counts as none. A
// thread owns eight columns (or one) of a token. Bound by HBM: 16384 tokens, 8 rows of
// 2048 each, 157 us (5.1 TB/s).
constexpr int kAtOnce = 8;

template <int DY, int DO, int V>
__global__ __launch_bounds__(256) void combine_kernel(RowsParams p) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t t = i / p.pieces;
  const int c = static_cast<int>(i - t * p.pieces) * V;
  if (t >= p.T) return;
  float acc[V];
  if (p.x) {
    Piece<DO, V> r;
    r.load(p.x, t * p.ldx + c);
#pragma unroll
    for (int q = 0; q < V; ++q) acc[q] = r.get(q);
  } else {
#pragma unroll
    for (int q = 0; q < V; ++q) acc[q] = 0.0f;
  }
  const int32_t* slots = p.slots + t * p.k;
  const float* weights = p.weights ? p.weights + t * p.k : nullptr;
  for (int j0 = 0; j0 < p.k; j0 += kAtOnce) {
    Piece<DY, V> y[kAtOnce];
    float w[kAtOnce];
    bool there[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int jj = min(j0 + j, p.k - 1);
      const int64_t s = slots[jj];
      there[j] = j0 + j < p.k && s >= 0 && s < p.R;
      w[j] = weights ? weights[jj] : 1.0f;
      if (there[j]) y[j].load(p.y, s * p.ldy + c);
      else y[j].zero();
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
      for (int q = 0; q < V; ++q) acc[q] += there[j] ? w[j] * y[j].get(q) : 0.0f;
  }
  store_piece<DO, V, false>(p.out, t * p.ldo + c, acc);
}

// W waves to a token: each of its rows is read once for its dot product and written
// once, x from the caches after its first reading. Bound by HBM: 4005 tokens, 2 rows of
// 3584 each, with the dots 41 us (4.2 TB/s), 16384 of 8 of 2048 272 (4.5) and 123 (4.9)
// without them.
template <int DX, int DY, int V, int W>
__global__ __launch_bounds__(256) void spread_kernel(RowsParams p) {
  __shared__ float smem[4][kAtOnce];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (4 / W) + (W == 4 ? 0 : wave);
  if (t >= p.T) return;  // (W 4: the whole block)
  const int first = W == 4 ? static_cast<int>(threadIdx.x) : lane;
  const int32_t* slots = p.slots + t * p.k;
  for (int j0 = 0; j0 < p.k; j0 += kAtOnce) {
    int64_t s[kAtOnce];
    float w[kAtOnce], dot[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int jj = min(j0 + j, p.k - 1);
      s[j] = slots[jj];
      if (j0 + j >= p.k || s[j] >= p.R) s[j] = -1;
      w[j] = p.weights ? p.weights[t * p.k + jj] : 1.0f;
      dot[j] = 0.0f;
    }
    for (int i = first; i < p.pieces; i += 64 * W) {
      const int c = i * V;
      Piece<DX, V> x;
      x.load(p.x, t * p.ldx + c);
      Piece<DY, V> y[kAtOnce];
      if (p.dweights) {
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          if (s[j] >= 0) y[j].load(p.y_old, s[j] * p.ldyo + c);
          else y[j].zero();
        }
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
          for (int q = 0; q < V; ++q) dot[j] += x.get(q) * y[j].get(q);
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        if (s[j] < 0) continue;
        float o[V];
#pragma unroll
        for (int q = 0; q < V; ++q) o[q] = w[j] * x.get(q);
        store_piece<DY, V, false>(p.y, s[j] * p.ldy + c, o);
      }
    }
    if (p.dweights) {
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) dot[j] = wave_sum(dot[j]);
      if constexpr (W == 4) {
        if (lane == 0) {
#pragma unroll
          for (int j = 0; j < kAtOnce; ++j) smem[wave][j] = dot[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) dot[j] = (smem[0][j] + smem[1][j]) + (smem[2][j] + smem[3][j]);
        __syncthreads();
      }
      if (first == 0) {
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
          if (j0 + j < p.k) p.dweights[t * p.k + j0 + j] = s[j] >= 0 ? dot[j] : 0.0f;
      }
    }
  }
}

int route_blocks(int64_t T, int64_t* chunk_out) {
  // Multiples of 64 tokens (a pass of a block with 16 lanes each), for at most 256
  // blocks; up to 128 tokens one block, which needs no second kernel (128 tokens of 128
  // experts by two blocks 11.9 us, one 9.5).
  const int64_t chunk = T <= 128 ? 128 : ((T + 255) / 256 + 63) / 64 * 64;
  *chunk_out = chunk;
  const int64_t n = (T + chunk - 1) / chunk;
  return static_cast<int>(n > 0 ? n : 1);
}

int check_route(const char* fn, int dtype, int64_t ldz, int64_t T, int64_t E, int64_t k, const void* z) {
  if (T < 0 || E <= 0 || k <= 0) return fail(MR_EINVAL, "%s: no experts to choose or from, or a negative size", fn);
  if (!valid_dtype(dtype)) return fail(MR_EINVAL, "%s: bad dtype %d", fn, dtype);
  if (k > E || k > kMaxTop || E > kMaxExperts)
    return fail(MR_EINVAL, "%s: at most %d of at most %d experts, no more than there are (%lld of %lld)", fn, kMaxTop,
                kMaxExperts, static_cast<long long>(k), static_cast<long long>(E));
  // (the last block's chunk, of at most 2^23 tokens in 64s, may end past T and must end within 31 bits)
  if (T > 0x7fffffff / k || T > 0x80000000ll - (1 << 14)) return fail(MR_EINVAL, "%s: too many rows", fn);
  if (T > 0 && ldz < E) return fail(MR_EINVAL, "%s: a leading dimension is smaller than its row", fn);
  if (reinterpret_cast<uintptr_t>(z) % dtype_bytes(dtype))
    return fail(MR_EINVAL, "%s: a pointer is not aligned to its elements", fn);
  return MR_OK;
}

bool whole_runs(const void* p, int64_t ld, int64_t E, int es) {
  return E % 4 == 0 && ld % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (4 * es) == 0;
}

// Lanes to a token: one for each entry, with at most 16 logits each.
int route_lanes(int64_t E, int64_t k) {
  if (k <= 16 && E <= 256) return 16;
  return k <= 32 && E <= 512 ? 32 : 64;
}

#define MR_ROUTE_V(DT, L, CALL)                           \
  do {                                                    \
    if (E <= 4 * L) CALL(DT, L, 4);                       \
    else if (L == 64 || E <= 8 * L) CALL(DT, L, 8);       \
    else CALL(DT, L, (L == 64 ? 8 : 16));                 \
  } while (0)
#define MR_ROUTE_L(DT, CALL)                       \
  do {                                             \
    if (lanes == 16) MR_ROUTE_V(DT, 16, CALL);     \
    else if (lanes == 32) MR_ROUTE_V(DT, 32, CALL); \
    else MR_ROUTE_V(DT, 64, CALL);                 \
  } while (0)
#define MR_ROUTE_CASES(CALL)                         \
  do {                                               \
    if (dtype == MR_F32) MR_ROUTE_L(MR_F32, CALL);   \
    else if (dtype == MR_BF16) MR_ROUTE_L(MR_BF16, CALL); \
    else MR_ROUTE_L(MR_F16, CALL);                   \
  } while (0)

int64_t rows_bytes(int64_t n, int64_t ld, int64_t H, int es) { return n > 0 ? ((n - 1) * ld + H) * es : 0; }

struct Bytes {
  const void* p;
  int64_t n;
};
template <int NW, int NR>
bool clash(const Bytes (&w)[NW], const Bytes (&r)[NR]) {
  for (int a = 0; a < NW; ++a) {
    if (!w[a].p || w[a].n <= 0) continue;
    for (int b = 0; b < NR; ++b)
      if (r[b].p && r[b].n > 0 && overlap(w[a].p, w[a].n, r[b].p, r[b].n)) return true;
    for (int b = a + 1; b < NW; ++b)
      if (w[b].p && w[b].n > 0 && overlap(w[a].p, w[a].n, w[b].p, w[b].n)) return true;
  }
  return false;
}

bool on4(const void* a, const void* b = nullptr, const void* c = nullptr, const void* d = nullptr) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) |
           reinterpret_cast<uintptr_t>(d)) & 3) == 0;
}

bool vector_rows(const void* p, int64_t ld, int es) { return !p || (aligned16(p) && ld * es % 16 == 0); }

int check_rows(const char* fn, int64_t T, int64_t k, int64_t R, int64_t H) {
  if (T < 0 || k <= 0 || R < 0 || H < 0) return fail(MR_EINVAL, "%s: no experts, or a negative size", fn);
  if (H > 0x7fffffff || T > 0x7fffffff / k || R > 0x7fffffff) return fail(MR_EINVAL, "%s: too large", fn);
  return MR_OK;
}

}  // namespace
}  // namespace mr

extern "C" {

size_t mr_route_workspace_bytes(int64_t T, int64_t E) {
  int64_t chunk;
  const int blocks = mr::route_blocks(T > 0 ? T : 0, &chunk);
  return blocks > 1 && E > 0 ? static_cast<size_t>(blocks) * E * 4 : 0;
}

int mr_route_experts(const void* logits, int dtype, int64_t ld, int64_t T, int64_t E, int64_t k, int normalize,
                     float scale, float* weights, int32_t* ids, int32_t* offsets, int32_t* slots, int32_t* rows,
                     void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mr;
  clear_error();
  const char* fn = "mr_route_experts";
  if (const int rc = check_route(fn, dtype, ld, T, E, k, logits)) return rc;
  if (T > 0 && (!logits || !weights || !ids)) return fail(MR_EINVAL, "%s: null pointer", fn);
  if (!offsets ? slots || rows : T > 0 && (!slots || !rows))
    return fail(MR_EINVAL, "%s: offsets, slots and rows come together", fn);
  if (T == 0 && !offsets) return MR_OK;
  if (!on4(weights, ids) || !on4(offsets, slots, rows, workspace))
    return fail(MR_EINVAL, "%s: a pointer is not aligned to its elements", fn);
  const size_t need = offsets ? mr_route_workspace_bytes(T, E) : 0;
  if (need && (!workspace || workspace_bytes < need)) return fail(MR_EINVAL, "%s: %zu bytes of workspace are needed", fn, need);
  {
    const int64_t n = T * k * 4;
    const Bytes w[6] = {{weights, n}, {ids, n}, {offsets, (E + 1) * 4}, {slots, n}, {rows, n},
                        {need ? workspace : nullptr, static_cast<int64_t>(need)}};
    const Bytes r[1] = {{logits, rows_bytes(T, ld, E, dtype_bytes(dtype))}};
    if (clash(w, r)) return fail(MR_EINVAL, "%s: outputs and the workspace must not overlap the logits or each other", fn);
  }
  RouteParams p{};
  int64_t chunk;
  p.blocks = route_blocks(T, &chunk);
  p.chunk = static_cast<int>(chunk);
  p.z = logits;
  p.ldz = ld;
  p.T = static_cast<int>(T);
  p.E = static_cast<int>(E);
  p.k = static_cast<int>(k);
  p.normalize = normalize != 0;
  p.whole = whole_runs(logits, ld, E, dtype_bytes(dtype));
  p.scale = scale;
  p.weights = weights;
  p.ids = ids;
  p.offsets = offsets;
  p.slots = slots;
  p.rows = rows;
  p.counts = static_cast<int32_t*>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(p.blocks), block(kRouteThreads);
  const size_t lds = route_lds(E);
  const int lanes = route_lanes(E, k);
#define MR_CHOOSE(DT, L, V) hipLaunchKernelGGL((route_choose<DT, L, V>), grid, block, lds, s, p)
  MR_ROUTE_CASES(MR_CHOOSE);
#undef MR_CHOOSE
  MR_LAUNCH_CHECK(fn);
  if (offsets && p.blocks > 1) {
    hipLaunchKernelGGL(route_place, grid, block, lds, s, p);
    MR_LAUNCH_CHECK(fn);
  }
  return MR_OK;
}

int mr_route_experts_bwd(const float* dweights, const void* logits, int dtype, int64_t ld, const int32_t* ids, int64_t T,
                         int64_t E, int64_t k, int normalize, float scale, void* dlogits, int64_t lddz, void* stream) {
  using namespace mr;
  clear_error();
  const char* fn = "mr_route_experts_bwd";
  if (const int rc = check_route(fn, dtype, ld, T, E, k, logits)) return rc;
  if (T == 0) return MR_OK;
  if (!dweights || !logits || !ids || !dlogits) return fail(MR_EINVAL, "%s: null pointer", fn);
  if (lddz < E) return fail(MR_EINVAL, "%s: a leading dimension is smaller than its row", fn);
  const int es = dtype_bytes(dtype);
  if (!on4(dweights, ids) || reinterpret_cast<uintptr_t>(dlogits) % es)
    return fail(MR_EINVAL, "%s: a pointer is not aligned to its elements", fn);
  {
    const bool in_place = dlogits == logits && lddz == ld;
    const Bytes w[1] = {{dlogits, rows_bytes(T, lddz, E, es)}};
    const Bytes r[3] = {{in_place ? nullptr : logits, rows_bytes(T, ld, E, es)}, {dweights, T * k * 4}, {ids, T * k * 4}};
    if (clash(w, r)) return fail(MR_EINVAL, "%s: dlogits may be the logits, and overlaps nothing else", fn);
  }
  RouteBwdParams p{};
  p.f.z = logits;
  p.f.ldz = ld;
  p.f.T = static_cast<int>(T);
  p.f.E = static_cast<int>(E);
  p.f.k = static_cast<int>(k);
  p.f.normalize = normalize != 0;
  p.f.whole = whole_runs(logits, ld, E, es) && whole_runs(dlogits, lddz, E, es);
  p.f.scale = scale;
  p.f.ids = const_cast<int32_t*>(ids);
  p.dw = dweights;
  p.dz = dlogits;
  p.lddz = lddz;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int lanes = route_lanes(E, k);
  const int64_t blocks = (T * lanes + 255) / 256;
  if (too_many_blocks(blocks, 256)) return fail(MR_EINVAL, "%s: too many rows", fn);
  const dim3 grid(static_cast<unsigned>(blocks)), block(256);
#define MR_BACK(DT, L, V) hipLaunchKernelGGL((route_bwd<DT, L, V>), grid, block, 0, s, p)
  MR_ROUTE_CASES(MR_BACK);
#undef MR_BACK
  MR_LAUNCH_CHECK(fn);
  return MR_OK;
}

int mr_combine_experts(const void* y, int y_dtype, int64_t ldy, int64_t R, const int32_t* slots, const float* weights,
                       int64_t T, int64_t k, int64_t H, const void* resid, int64_t ldr, void* out, int out_dtype,
                       int64_t ldo, void* stream) {
  using namespace mr;
  clear_error();
  const char* fn = "mr_combine_experts";
  if (const int rc = check_rows(fn, T, k, R, H)) return rc;
  if ((y_dtype != MR_F32 && y_dtype != MR_BF16) || (out_dtype != MR_F32 && out_dtype != MR_BF16))
    return fail(MR_EINVAL, "%s: rows are fp32 or bf16", fn);
  if (T == 0 || H == 0) return MR_OK;
  if (!slots || !out || (!y && R)) return fail(MR_EINVAL, "%s: null pointer", fn);
  const int ey = dtype_bytes(y_dtype), eo = dtype_bytes(out_dtype);
  if ((R > 0 && ldy < H) || ldo < H || (resid && ldr < H))
    return fail(MR_EINVAL, "%s: a leading dimension is smaller than its row", fn);
  if (reinterpret_cast<uintptr_t>(y) % ey || (reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(resid)) % eo ||
      !on4(slots, weights))
    return fail(MR_EINVAL, "%s: a pointer is not aligned to its elements", fn);
  {
    const bool in_place = out == resid && ldo == ldr;
    const Bytes w[1] = {{out, rows_bytes(T, ldo, H, eo)}};
    const Bytes r[4] = {{y, rows_bytes(R, ldy, H, ey)}, {in_place ? nullptr : resid, rows_bytes(T, ldr, H, eo)},
                        {slots, T * k * 4}, {weights, T * k * 4}};
    if (clash(w, r)) return fail(MR_EINVAL, "%s: out may be resid, and overlaps nothing else", fn);
  }
  RowsParams p{};
  p.x = resid;
  p.ldx = ldr;
  p.y = const_cast<void*>(y);
  p.ldy = ldy;
  p.R = R;
  p.slots = slots;
  p.weights = weights;
  p.out = out;
  p.ldo = ldo;
  p.T = T;
  p.H = static_cast<int>(H);
  p.k = static_cast<int>(k);
  const bool vec = H % 8 == 0 && vector_rows(y, ldy, ey) && vector_rows(resid, ldr, eo) && vector_rows(out, ldo, eo);
  p.pieces = static_cast<int>(vec ? H / 8 : H);
  const int64_t blocks = (T * p.pieces + 255) / 256;
  if (too_many_blocks(blocks, 256)) return fail(MR_EINVAL, "%s: too large", fn);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(blocks)), block(256);
#define MR_COMBINE(DY, DO)                                                                        \
  do {                                                                                            \
    if (vec) hipLaunchKernelGGL((combine_kernel<DY, DO, 8>), grid, block, 0, s, p);               \
    else hipLaunchKernelGGL((combine_kernel<DY, DO, 1>), grid, block, 0, s, p);                   \
  } while (0)
  if (y_dtype == MR_BF16) {
    if (out_dtype == MR_F32) MR_COMBINE(MR_BF16, MR_F32);
    else MR_COMBINE(MR_BF16, MR_BF16);
  } else {
    if (out_dtype == MR_F32) MR_COMBINE(MR_F32, MR_F32);
    else MR_COMBINE(MR_F32, MR_BF16);
  }
#undef MR_COMBINE
  MR_LAUNCH_CHECK(fn);
  return MR_OK;
}

int mr_spread_experts(const void* x, int x_dtype, int64_t ldx, const int32_t* slots, const float* weights, int64_t T,
                      int64_t k, int64_t H, void* out, int out_dtype, int64_t ldo, int64_t R, const void* y, int64_t ldy,
                      float* dweights, void* stream) {
  using namespace mr;
  clear_error();
  const char* fn = "mr_spread_experts";
  if (const int rc = check_rows(fn, T, k, R, H)) return rc;
  if (H > 0x7fffffff - 256) return fail(MR_EINVAL, "%s: too large", fn);  // (a block's steps over the columns: 31 bits)
  if ((x_dtype != MR_F32 && x_dtype != MR_BF16) || (out_dtype != MR_F32 && out_dtype != MR_BF16))
    return fail(MR_EINVAL, "%s: rows are fp32 or bf16", fn);
  if (T == 0 || (H == 0 && !dweights)) return MR_OK;
  if (!dweights != !y && R) return fail(MR_EINVAL, "%s: the weights' gradients and the rows they multiply come together", fn);
  if (H == 0) return fail(MR_EINVAL, "%s: no columns to sum dweights over", fn);
  if (!x || !slots || (!out && R)) return fail(MR_EINVAL, "%s: null pointer", fn);
  const int ex = dtype_bytes(x_dtype), eo = dtype_bytes(out_dtype);
  if (ldx < H || (R > 0 && (ldo < H || (y && ldy < H))))
    return fail(MR_EINVAL, "%s: a leading dimension is smaller than its row", fn);
  if (reinterpret_cast<uintptr_t>(x) % ex || (reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(y)) % eo ||
      !on4(slots, weights, dweights))
    return fail(MR_EINVAL, "%s: a pointer is not aligned to its elements", fn);
  {
    const bool in_place = out == y && ldo == ldy;
    const Bytes w[2] = {{out, rows_bytes(R, ldo, H, eo)}, {dweights, T * k * 4}};
    const Bytes r[4] = {{x, rows_bytes(T, ldx, H, ex)}, {in_place ? nullptr : y, rows_bytes(R, ldy, H, eo)},
                        {slots, T * k * 4}, {weights, T * k * 4}};
    if (clash(w, r)) return fail(MR_EINVAL, "%s: out may be y; outputs overlap nothing else", fn);
  }
  RowsParams p{};
  p.x = x;
  p.ldx = ldx;
  p.y = out;
  p.ldy = ldo;
  p.y_old = y;
  p.ldyo = ldy;
  p.R = R;
  p.slots = slots;
  p.weights = weights;
  p.dweights = dweights;
  p.T = T;
  p.H = static_cast<int>(H);
  p.k = static_cast<int>(k);
  const bool vec = H % 8 == 0 && vector_rows(x, ldx, ex) && vector_rows(out, ldo, eo) && vector_rows(y, ldy, eo);
  p.pieces = static_cast<int>(vec ? H / 8 : H);
  // A wave to a token where that fills the card twice over, else a block.
  const bool one = T >= 4096 || p.pieces <= 64;
  const int64_t blocks = one ? (T + 3) / 4 : T;
  if (too_many_blocks(blocks, 256)) return fail(MR_EINVAL, "%s: too large", fn);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(blocks)), block(256);
#define MR_SPREAD(DX, DY)                                                                           \
  do {                                                                                              \
    if (vec && one) hipLaunchKernelGGL((spread_kernel<DX, DY, 8, 1>), grid, block, 0, s, p);        \
    else if (vec) hipLaunchKernelGGL((spread_kernel<DX, DY, 8, 4>), grid, block, 0, s, p);          \
    else if (one) hipLaunchKernelGGL((spread_kernel<DX, DY, 1, 1>), grid, block, 0, s, p);          \
    else hipLaunchKernelGGL((spread_kernel<DX, DY, 1, 4>), grid, block, 0, s, p);                   \
  } while (0)
  if (x_dtype == MR_BF16) {
    if (out_dtype == MR_F32) MR_SPREAD(MR_BF16, MR_F32);
    else MR_SPREAD(MR_BF16, MR_BF16);
  } else {
    if (out_dtype == MR_F32) MR_SPREAD(MR_F32, MR_F32);
    else MR_SPREAD(MR_F32, MR_BF16);
  }
#undef MR_SPREAD
  MR_LAUNCH_CHECK(fn);
  return MR_OK;
}

}  // extern "C"
