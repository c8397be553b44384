// A teacher's top logits and the distillation loss against them, for gfx950.
//
// Top logits: the k largest of a row in order, ties to the lower index, and the
// row's log-sum-exp at a temperature. The teacher's list of a position.
//
// Distillation: with student logits z, u = z / T, p = softmax(u), and the
// teacher's list t_j at ids S,
//   whole = false (the teacher's log-sum-exp L at T is given):
//     q_j = exp(t_j / T - L), q_R = max(0, 1 - sum q_j): the vocabulary off S is
//     one outcome more, of probability p_R = sum_{i not in S} p_i;
//   whole = true: q = softmax(t / T) over the list, q_R = 0;
//   loss = sum_j q_j (log q_j - log p_j) + q_R (log q_R - log p_R),
//   dloss/dz_i = (p_i Q - q_i) / T on S,  p_i (Q - q_R / p_R) / T off S,  Q = sum q + q_R.
//
// Both read rows of a vocabulary and are bound by memory. Top logits and the loss
// alone read a row once; with the gradient a row is read once as far as half a CU's
// registers and LDS hold it, beyond that twice in part, past 20,480 pieces of 16 bytes
// twice, and its gradient is written once. Row sums run in fp32; the list's terms,
// whose differences are the loss, and 1 - sum q in fp64.
#include <cmath>
#include <limits>
#include <type_traits>

#include "mr_common.h"

namespace mr {
namespace {

constexpr float kInf = __builtin_inff(), kMaxFloat = 3.4028234663852886e38f;
constexpr int kMaxTop = 1024;

// 16 bytes at any element; nt: past the caches, of what is read once.
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ uint4 ld16(const uint8_t* p) {
  uint4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
__device__ __forceinline__ uint4 ld16nt(const uint8_t* p) {
  const u32x4u v = __builtin_nontemporal_load(reinterpret_cast<const u32x4u*>(p));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// Elements of a 16-byte piece of type DT, widened.
template <int DT>
constexpr int kPiece = DT == MR_F32 ? 4 : 8;

template <int DT>
__device__ __forceinline__ void widen(uint4 r, float (&v)[kPiece<DT>]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (DT == MR_F32) {
      v[k] = __uint_as_float(w[k]);
    } else if constexpr (DT == MR_BF16) {
      v[2 * k] = __uint_as_float(w[k] << 16);
      v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    } else {
      v[2 * k] = f16_to_f32(static_cast<uint16_t>(w[k] & 0xffffu));
      v[2 * k + 1] = f16_to_f32(static_cast<uint16_t>(w[k] >> 16));
    }
  }
}

template <int DT>
__device__ __forceinline__ uint4 narrow(const float (&v)[kPiece<DT>]) {
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (DT == MR_F32) w[k] = __float_as_uint(v[k]);
    else if constexpr (DT == MR_BF16) w[k] = pack_bf16x2(v[2 * k], v[2 * k + 1]);
    else w[k] = static_cast<uint32_t>(f32_to_f16(v[2 * k])) | (static_cast<uint32_t>(f32_to_f16(v[2 * k + 1])) << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Minus infinity in every element: no part in a maximum or a sum.
template <int DT>
__device__ __forceinline__ uint4 no_piece() {
  constexpr uint32_t w = DT == MR_F32 ? 0xff800000u : DT == MR_BF16 ? 0xff80ff80u : 0xfc00fc00u;
  return make_uint4(w, w, w, w);
}

// The listed or left out ones of a piece at minus infinity, a bit each.
template <int DT>
__device__ __forceinline__ void take_out(uint4& q, uint32_t bits) {
  uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (DT == MR_F32) {
      if (bits >> k & 1) w[k] = 0xff800000u;
    } else {
      constexpr uint32_t inf = DT == MR_BF16 ? 0xff80u : 0xfc00u;
      if (bits >> (2 * k) & 1) w[k] = (w[k] & 0xffff0000u) | inf;
      if (bits >> (2 * k + 1) & 1) w[k] = (w[k] & 0xffffu) | (inf << 16);
    }
  }
  q = make_uint4(w[0], w[1], w[2], w[3]);
}

// Piece i of a row of V >= E elements, any i: what no earlier piece has of the 16
// bytes that start at its first element or end the row, whichever is sooner; the
// rest is minus infinity. The load is whole and without a branch (a branch around
// a load makes each wait for the last).
template <int DT, bool NT = false>
__device__ __forceinline__ uint4 piece_bytes(const uint8_t* row, int64_t i, int64_t V) {
  constexpr int E = kPiece<DT>, ES = 16 / E;
  const uint8_t* at = row + min(i * E, V - E) * ES;
  return NT ? ld16nt(at) : ld16(at);
}
template <int DT>
__device__ __forceinline__ uint32_t piece_drop(int64_t i, int64_t V) {  // bits of the elements that are not the piece's
  constexpr int E = kPiece<DT>;
  const int64_t over = i * E - (V - E);
  return over <= 0 ? 0u : (1u << (over < E ? static_cast<int>(over) : E)) - 1;
}

// The same of a row shorter than a piece, element by element.
template <int DT>
__device__ __forceinline__ uint4 short_row(const uint8_t* row, int64_t V) {
  constexpr int E = kPiece<DT>, ES = 16 / E;
  uint4 r = no_piece<DT>();
  uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int k = 0; k < E - 1; ++k) {
    if (k >= V) continue;
    if constexpr (ES == 4) {
      w[k] = reinterpret_cast<const uint32_t*>(row)[k];
    } else {
      const uint32_t x = reinterpret_cast<const uint16_t*>(row)[k];
      w[k >> 1] = (k & 1) ? (w[k >> 1] & 0xffffu) | (x << 16) : (w[k >> 1] & 0xffff0000u) | x;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// exp(d / T) for d = x - max: log2(e) / T in two floats, so that the exponent's
// error is its rounding alone (the constant's own, up to 2^-25 of it, has one
// sign and would add up over a row). Below 2^-126 the result is zero.
struct ExpScale {
  float hi, lo;
};
__device__ __forceinline__ float exp_t(float d, ExpScale c) {
  return __builtin_amdgcn_exp2f(__builtin_fmaf(d, c.hi, d * c.lo));
}

// A value that all lanes share, in a scalar register.
__device__ __forceinline__ float uniform(float x) {
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x)));
}

// Past 2^24 powers of two a float's step is one power or more, and v hi - base (base: max hi, rounded) is off
// zero at the maximum itself by as much: exponentials of a few hundred past 2^30. There, far from zero, terms are
// formed of differences (exp_t), or, of 16-bit logits, whose steps are then 2^13 powers and leave of all terms
// those at the maximum, with a log2(e) / T of 12 bits, whose product with it is exact.
constexpr float kFar = 0x1p24f;
__device__ __forceinline__ bool is_far(float about, ExpScale c) {
  const float x = __builtin_fabsf(about * c.hi);
  return x > kFar && x < kInf;
}
template <int DT>
__device__ __forceinline__ ExpScale scale_at(float about, ExpScale c) {
  if constexpr (DT != MR_F32) {
    const uint32_t hi = __float_as_uint(c.hi);
    c.hi = uniform(__uint_as_float(is_far(about, c) ? hi & 0xfffff000u : hi));
  }
  return c;
}
// The base of a sum about a far maximum, in powers of two.
__device__ __forceinline__ double far_base(float about, ExpScale c) {
  return static_cast<double>(about) * (static_cast<double>(c.hi) + c.lo);
}

// A piece's gradient: its terms as the sum had them, 2^(v hi - b), times g; in fp32
// to its precision, about `about`.
template <int DT>
__device__ __forceinline__ uint4 gradient_piece(uint4 q, float about, float b, float g, ExpScale c) {
  constexpr int E = kPiece<DT>;
  float v[E];
  widen<DT>(q, v);
#pragma unroll
  for (int k = 0; k < E; ++k)
    v[k] = (DT == MR_F32 ? exp_t(v[k] - about, c) : __builtin_amdgcn_exp2f(__builtin_fmaf(v[k], c.hi, b))) * g;
  return narrow<DT>(v);
}

// Temperatures whose log2(e) / T leaves room for masked logits and for its low part.
constexpr double kMinTemperature = 1.0 / 1024, kMaxTemperature = 1024.0;

ExpScale exp_scale(double temperature) {
  // hi from below and lo above zero: minus infinity times either is minus infinity
  const double c = 1.4426950408889634073599 / temperature;
  float hi = static_cast<float>(c);
  if (hi > c) hi = std::nextafter(hi, 0.0f);
  const float lo = static_cast<float>(c - hi);
  return {hi, lo > 0.0f ? lo : std::numeric_limits<float>::min()};
}

__device__ __forceinline__ float wave_max(float x) {
  for (int off = 32; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, 64));
  return x;
}
template <typename T>
__device__ __forceinline__ T wave_sum(T x) {
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

// The maximum or the sum of W waves' values, to every lane. (A lane reads one of
// them: all W in every lane's registers at once, for eight such reductions,
// made the held rows spill.)
template <int W>
__device__ __forceinline__ float waves_max(const float* v) {
  float x = v[threadIdx.x % W];
  for (int off = W / 2; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, 64));
  return x;
}
template <int W, typename T>
__device__ __forceinline__ T waves_sum(const T* v) {
  T x = v[threadIdx.x % W];
  for (int off = W / 2; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

// A logit at or below this has no part in a sum: masks write the types' lowest
// values, whose exponents are no floats.
constexpr float kMasked = -1e37f;

// A sum and its mean's terms under a greater base. What was summed among masks far from zero can be infinite
// (is_far), and times zero no number: nothing is left of it. NaN stays.
__device__ __forceinline__ void rebase(float& s, float& ve, float& e, float f) {
  if (f == 0.0f) {
    if (s == s) s = 0.0f;
    ve = e = 0.0f;
  }
  s *= f;
  ve *= f;
  e *= f;
}

// The mean of v over a sum's terms, from one in E of them: v_e their sum of v, e of their
// terms. Where they have under half of their share of the sum, peaks lie among the
// others, and what these have too much lies at `peak`. (By the mean of the rest alone a
// peak 80 above it left the sum's logarithm 4e-6 off.)
template <int E>
__device__ __forceinline__ float mean_logit(float sum, float v_e, float e, float peak) {
  const float more = sum - E * e;
  return more > 0.5f * sum ? (E * v_e + more * peak) / (E * e + more) : v_e / e;
}

// A running sum of exp(v / T), as s 2^base: base is max hi, so a term is one fused
// multiply-add and the exponential, 2^(v hi - base). What hi lacks of log2(e) / T
// comes back at the end, to first order, with the mean of v (from one in E of the terms).
struct RunningSum {
  float max = -kInf, base = 0.0f, s = 0.0f, ve = 0.0f, e = 0.0f;

  template <int DT, int U>
  __device__ __forceinline__ void add(const uint4 (&r)[U], float mx, ExpScale c) {
    constexpr int E = kPiece<DT>;
    if (mx > max) {
      if (mx > kMasked) {
        // (a product past the floats is their end: an exponential above it overflows, as it should)
        const float grown = clampf(mx * c.hi, -kMaxFloat, kMaxFloat), f = max > kMasked ? __builtin_amdgcn_exp2f(base - grown) : 1.0f;
        base = grown;
        rebase(s, ve, e, f);
      }
      max = mx;
    }
    const float b = -base;
    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float v[E];
      widen<DT>(r[j], v);
#pragma unroll
      for (int k = 0; k < E; k += 2) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(v[k], c.hi, b));
        if (k == 0) {
          ve = __builtin_fmaf(fmaxf(v[0], -1e30f), x, ve);
          e += x;
        }
        s0 += x;
        s1 += __builtin_amdgcn_exp2f(__builtin_fmaf(v[k + 1], c.hi, b));
      }
    }
    s += s0 + s1;
  }

  template <int W>
  struct Shared {
    float max[W], base[W], s[W], ve[W], e[W];
  };
  // The wave's into the block's, before a barrier.
  template <int W>
  __device__ __forceinline__ void publish(Shared<W>& sh) {
    const float about = wave_max(max > kMasked ? base : -kInf), f = max > kMasked ? __builtin_amdgcn_exp2f(base - about) : 1.0f;
    max = wave_max(max);
    rebase(s, ve, e, f);
    s = wave_sum(s);
    ve = wave_sum(ve);
    e = wave_sum(e);
    if ((threadIdx.x & 63) == 0) {
      const int w = threadIdx.x >> 6;
      sh.max[w] = max;
      sh.base[w] = about;
      sh.s[w] = s;
      sh.ve[w] = ve;
      sh.e[w] = e;
    }
  }
};

// The block's sum: sum 2^exponent, and the maximum, on every thread.
template <int W, int E>
struct BlockSum {
  double sum, exponent;
  float max;
  __device__ __forceinline__ BlockSum(const RunningSum::Shared<W>& sh, ExpScale c) {
    const int w = threadIdx.x % W;
    max = waves_max<W>(sh.max);
    const float about = waves_max<W>(sh.base), f = sh.base[w] == -kInf ? 1.0f : __builtin_amdgcn_exp2f(sh.base[w] - about);
    float s = sh.s[w], v = sh.ve[w], n = sh.e[w];
    rebase(s, v, n, f);
    sum = static_cast<double>(s);
    for (int off = W / 2; off > 0; off >>= 1) {
      sum += __shfl_xor(sum, off, 64);
      v += __shfl_xor(v, off, 64);
      n += __shfl_xor(n, off, 64);
    }
    // (far from zero the mean of v, which ends at -1e30, is the maximum to a few steps of 2^-24)
    const float mean = n > 0.0f && v < kInf && v > -kInf && !is_far(max, c) ? mean_logit<E>(static_cast<float>(sum), v, n, max) : max;
    exponent = about == -kInf ? 0.0 : static_cast<double>(about) + static_cast<double>(c.lo) * mean;
  }
};

// ------------------------------------------------------------------ top logits --

// A float's place in the order of values: greater keys are greater, the zeros
// are equal, NaN is above all. Zero is no float's key.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k == 0xffffffffu ? 0x7fc00000u : k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

constexpr int kCandidates = 2048;

struct TopParams {
  const void* x;
  int64_t ld, V;
  int k;
  ExpScale c;
  double temperature;
  float* values;
  int32_t* ids;
  float* lse;
};

// One workgroup per row, which it reads once. A thread keeps the largest of its
// even and of its odd pieces: the k-th largest of these 2 THREADS maxima (of
// their keys' upper halves) cannot exceed the row's k-th largest logit, and few
// logits reach it. Those lie in the pieces of the maxima that reach it, which
// are read again (a piece or two per thread, from cache) and filtered into a
// list in LDS that is then ordered whole. A row with more candidates than the
// list holds (many ties), a NaN or an infinity takes the radix selection.
template <int DT, int THREADS>
__global__ __launch_bounds__(THREADS, 8) void top_rows(TopParams p) {
  constexpr int E = kPiece<DT>, ES = 16 / E, W = THREADS / 64, U = 4;
  __shared__ unsigned long long list[kCandidates];
  __shared__ int owners[2 * THREADS];
  __shared__ RunningSum::Shared<W> s_sum;
  __shared__ int counts[2][4][W];
  __shared__ int n_owners, n_list;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x, V = p.V;
  const uint8_t* x = static_cast<const uint8_t*>(p.x) + row * p.ld * ES;
  const int64_t pieces = (V + E - 1) / E;
  if (tid == 0) n_owners = n_list = 0;

  float top[2] = {-kInf, -kInf};
  const bool has[2] = {tid < pieces, tid + THREADS < pieces};
  RunningSum running;
  auto add_up = [&](const uint4(&r)[U]) __attribute__((always_inline)) {
    float mx[2] = {-kInf, -kInf};
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float v[E];
      widen<DT>(r[j], v);
#pragma unroll
      for (int k = 0; k < E; ++k) mx[j & 1] = fmaxf(mx[j & 1], v[k]);
    }
    top[0] = fmaxf(top[0], mx[0]);
    top[1] = fmaxf(top[1], mx[1]);
    running.add<DT, U>(r, fmaxf(mx[0], mx[1]), p.c);
  };
  if (V >= E) {
    for (int64_t i0 = tid; i0 < pieces; i0 += U * THREADS) {
      uint4 r[U];
#pragma unroll
      for (int j = 0; j < U; ++j) r[j] = piece_bytes<DT>(x, i0 + j * THREADS, V);
#pragma unroll
      for (int j = 0; j < U; ++j)
        if (const uint32_t drop = piece_drop<DT>(i0 + j * THREADS, V)) take_out<DT>(r[j], drop);
      add_up(r);
    }
  } else if (tid == 0) {
    uint4 r[U];
#pragma unroll
    for (int j = 0; j < U; ++j) r[j] = no_piece<DT>();
    r[0] = short_row<DT>(x, V);
    add_up(r);
  }
  running.publish<W>(s_sum);
  __syncthreads();
  bool odd;  // a NaN, an infinity, or no logit above the masks' values
  {
    const BlockSum<W, E> all(s_sum, p.c);
    odd = !(all.sum > 0.0 && all.sum < static_cast<double>(kInf) && all.max < kInf);
    // (odd: the maximum alone; a NaN is the list's first entry, which tells)
    if (tid == 0 && p.lse)
      p.lse[row] = static_cast<float>(odd ? all.max / p.temperature : 0.69314718055994530942 * all.exponent + log(all.sum));
  }

  // The largest 16-bit key that k of the maxima reach, two bits at a time. (Four bits
  // a time are fewer barriers and more ballots: 2044 rows of 151936 4 us slower. One
  // maximum a thread for short lists: twice the pieces to read again, 8 us slower.)
  uint32_t tau = 0;
  {
    const uint32_t k0 = has[0] ? order_key(top[0]) >> 16 : 0, k1 = has[1] ? order_key(top[1]) >> 16 : 0;
    for (int shift = 14, step = 0; shift >= 0; shift -= 2, ++step) {
      int(&cnt)[4][W] = counts[step & 1];
#pragma unroll
      for (uint32_t d = 1; d < 4; ++d) {
        const uint32_t t = tau | (d << shift);
        const int c = __popcll(__ballot(k0 >= t)) + __popcll(__ballot(k1 >= t));
        if (lane == 0) cnt[d][wave] = c;
      }
      __syncthreads();
      uint32_t best = 0;
#pragma unroll
      for (uint32_t d = 1; d < 4; ++d) {
        int c = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) c += cnt[d][w];
        if (c >= p.k) best = d;
      }
      tau |= best << shift;
    }
    if (!odd) {
      if (has[0] && k0 >= tau) owners[atomicAdd(&n_owners, 1)] = 2 * tid;
      if (has[1] && k1 >= tau) owners[atomicAdd(&n_owners, 1)] = 2 * tid + 1;
    }
  }
  __syncthreads();
  bool listed = false;
  if (!odd) {
    const int per = static_cast<int>((pieces + 2 * THREADS - 1) / (2 * THREADS));
    const int total = n_owners * per;
    for (int q = tid; q < total; q += THREADS) {
      const int o = q / per, j = q - o * per, own = owners[o];
      const int64_t i = (own >> 1) + static_cast<int64_t>(2 * j + (own & 1)) * THREADS;
      if (i >= pieces) continue;
      const int64_t start = V >= E ? min(i * E, V - E) : 0;
      const uint32_t drop = V >= E ? piece_drop<DT>(i, V) : 0xffffffffu << V;
      float v[E];
      widen<DT>(V >= E ? piece_bytes<DT>(x, i, V) : short_row<DT>(x, V), v);
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const uint32_t key = order_key(v[k]);
        if (key >> 16 >= tau && !(drop >> k & 1)) {
          const int at = atomicAdd(&n_list, 1);
          if (at < kCandidates)
            list[at] = (static_cast<unsigned long long>(key) << 32) | (0xffffffffu - static_cast<uint32_t>(start + k));
        }
      }
    }
    __syncthreads();
    listed = n_list <= kCandidates;
  }
  int n = n_list;
  if (!listed) {
    // Radix selection of the k-th largest key, a byte at a time from the top;
    // then every greater key and the first of the equal ones.
    __shared__ int hist[256];
    __shared__ uint32_t s_digit;
    __shared__ int s_need;
    uint32_t prefix = 0;
    int need = p.k;
    auto elem = [&](int64_t i) __attribute__((always_inline)) { return load_elem<DT>(x, i); };
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += THREADS) hist[i] = 0;
      __syncthreads();
      for (int64_t i0 = 0; i0 < V; i0 += THREADS) {
        const int64_t i = i0 + tid;
        const uint32_t key = i < V ? order_key(elem(i)) : 0;
        const bool in = i < V && (shift == 24 || key >> (shift + 8) == prefix);
        const uint32_t digit = (key >> shift) & 255u;
        // (lanes of one digit add once: rows of ties would queue at one counter)
        const unsigned long long live = __ballot(in);
        if (live) {
          const uint32_t first = __shfl(static_cast<int>(digit), __ffsll(live) - 1, 64);
          const unsigned long long same = __ballot(in && digit == first);
          if (in && digit != first) atomicAdd(&hist[digit], 1);
          if (lane == __ffsll(live) - 1) atomicAdd(&hist[first], __popcll(same));
        }
      }
      __syncthreads();
      if (tid == 0) {
        int above = 0, d = 255;
        while (above + hist[d] < need) above += hist[d--];
        s_digit = d;
        s_need = need - above;
      }
      __syncthreads();
      prefix = (prefix << 8) | s_digit;
      need = s_need;
    }
    if (tid == 0) {
      n_list = 0;
      n_owners = 0;  // of the equal keys
    }
    __syncthreads();
    for (int64_t i0 = 0; i0 < V; i0 += THREADS) {
      const int64_t i = i0 + tid;
      const uint32_t key = i < V ? order_key(elem(i)) : 0;
      const unsigned long long entry = (static_cast<unsigned long long>(key) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
      if (key > prefix) list[atomicAdd(&n_list, 1)] = entry;
      // equal keys in the order of their indexes
      const bool equal = i < V && key == prefix;
      const unsigned long long b = __ballot(equal);
      if (lane == 0) counts[0][0][wave] = __popcll(b);
      __syncthreads();
      int before = n_owners, all = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (w < wave) before += counts[0][0][w];
        all += counts[0][0][w];
      }
      before += __popcll(b & ((1ull << lane) - 1));
      if (equal && before < need) list[atomicAdd(&n_list, 1)] = entry;
      __syncthreads();
      if (tid == 0) n_owners += all;
      __syncthreads();
    }
    n = p.k;
  }
  __syncthreads();
  // The list in descending order. Short ones by counting, for each entry, those
  // above it; longer ones by a bitonic network.
  const int k_out = p.k;
  float* values = p.values + row * k_out;
  int32_t* ids = p.ids + row * k_out;
  auto emit = [&](int at, unsigned long long e) __attribute__((always_inline)) {
    values[at] = key_value(static_cast<uint32_t>(e >> 32));
    ids[at] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(e));
    if (at == 0 && odd && p.lse && static_cast<uint32_t>(e >> 32) == 0xffffffffu) p.lse[row] = __builtin_nanf("");
  };
  if (n <= 256) {
    int* rank = owners;
    for (int i = tid; i < 256; i += THREADS) rank[i] = 0;
    __syncthreads();
    // 64 entries a wave, the entries to compare with shared out among the waves
    const int groups = (n + 63) / 64, parts = W / groups > 0 ? W / groups : 1;
    for (int g = wave; g < groups * parts; g += W) {
      const int i = (g % groups) * 64 + lane, part = g / groups;
      const unsigned long long e = i < n ? list[i] : 0;
      int above = 0;
      for (int j = part; j < n; j += parts) above += list[j] > e;
      if (i < n) atomicAdd(&rank[i], above);
    }
    __syncthreads();
    for (int i = tid; i < n; i += THREADS)
      if (rank[i] < k_out) emit(rank[i], list[i]);
    return;
  }
  int size = 512;
  while (size < n) size *= 2;
  for (int i = n + tid; i < size; i += THREADS) list[i] = 0;
  __syncthreads();
  // (a wave's 64 pairs of strides up to 64 lie in 128 entries of its own, which its
  // LDS accesses, in order as they are, leave as the next stride needs them)
  for (int width = 2; width <= size; width *= 2)
    for (int stride = width / 2; stride > 0; stride /= 2) {
      if (stride > 64 || (stride == 64 && width > 128)) __syncthreads();
      for (int q = tid; q < size / 2; q += THREADS) {
        const int i = ((q & ~(stride - 1)) << 1) | (q & (stride - 1)), j = i + stride;
        const unsigned long long a = list[i], b = list[j];
        const bool down = (i & width) == 0;
        if ((a < b) == down) {
          list[i] = b;
          list[j] = a;
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
    }
  __syncthreads();
  for (int i = tid; i < k_out; i += THREADS) emit(i, list[i]);
}

// ---------------------------------------------------------------- distillation --

constexpr int kBitmapMaxV = 1 << 20;

struct DistillParams {
  const void* z;
  int64_t ldz;
  int V, k;
  const float* t;
  const int32_t* ids;
  const float* lse;  // null: the list is the whole distribution
  ExpScale c;
  double inv_t;
  float scale;
  float* row_loss;
  void* dz;  // null: no gradient
  int64_t ldd;
};

// The list of a row: entry e THREADS + tid is thread tid's. Ids and teacher's
// logits lie in LDS (behind the bitmap), a register each would not fit beside the
// held rows; the student's logits are gathered into registers.
template <int DT, int THREADS>
struct List {
  static constexpr int KE = kMaxTop / THREADS, W = THREADS / 64;
  using Raw = typename std::conditional<DT == MR_F32, uint32_t, uint16_t>::type;
  struct Shared {
    float t[W], z[W];
    int n[W];
    double q[W], a[W], s[W], rest[W];
  };
  int* ids;
  float* values;
  Raw raw[KE];  // the listed logits, as they lie in memory
  int n;        // entries; negative: a bad list
  float t_max, z_max, lse;
  double q_sum, a_sum, z_sum, shift;

  __device__ __forceinline__ List(uint32_t* lds, int k) : ids(reinterpret_cast<int*>(lds)), values(reinterpret_cast<float*>(lds + k)) {}
  // (not widened where it is loaded: that would wait for the row's pieces before it)
  __device__ __forceinline__ float z(int e) const {
    return DT == MR_F32 ? __uint_as_float(raw[e]) : DT == MR_BF16 ? bf16_to_f32(raw[e]) : f16_to_f32(raw[e]);
  }
  // f(e, id, t) for the thread's entries.
  template <typename F>
  __device__ __forceinline__ void each(const DistillParams& p, F f) const {
#pragma unroll
    for (int e = 0; e < KE; ++e) {
      const int j = e * THREADS + static_cast<int>(threadIdx.x);
      if (j < p.k) {
        const int id = ids[j];
        if (id >= 0) f(e, id, values[j]);
      }
    }
  }
  // The thread's entries, on their way while the row's loads are issued.
  struct Entries {
    int id[KE];
    float t[KE];
  };
  __device__ __forceinline__ Entries load(const DistillParams& p, int64_t row) {
    Entries x;
    lse = p.lse ? p.lse[row] : 0.0f;
#pragma unroll
    for (int e = 0; e < KE; ++e) {
      const int j = e * THREADS + static_cast<int>(threadIdx.x);
      x.id[e] = j < p.k ? p.ids[row * p.k + j] : -1;
      x.t[e] = j < p.k ? p.t[row * p.k + j] : 0.0f;
    }
    return x;
  }
  // Marks the entries in the bitmap (clear, behind a barrier), gathers their logits
  // and leaves the wave's counts and maximum in the block's. Entries past the
  // vocabulary or listed twice make the row a NaN.
  __device__ __forceinline__ void mark(const DistillParams& p, const Entries& x, const uint8_t* zrow, uint32_t* bitmap,
                                       Shared& s) {
    int count = 0;
    bool bad = false;
    float top = -kInf;
#pragma unroll
    for (int e = 0; e < KE; ++e) {
      raw[e] = 0;
      const int j = e * THREADS + static_cast<int>(threadIdx.x);
      int id = x.id[e];
      if (id >= p.V) {
        bad = true;
        id = -1;
      }
      if (j < p.k) {
        ids[j] = id;
        values[j] = x.t[e];
      }
      if (id < 0) continue;
      const uint32_t bit = 1u << (id & 31);
      if (atomicOr(&bitmap[id >> 5], bit) & bit) bad = true;
      raw[e] = reinterpret_cast<const Raw*>(zrow)[id];
      ++count;
      top = fmaxf(top, x.t[e]);
    }
    top = wave_max(top);
    count = __any(bad) ? -(1 << 20) : wave_sum(count);
    if ((threadIdx.x & 63) == 0) {
      s.t[threadIdx.x >> 6] = top;
      s.n[threadIdx.x >> 6] = count;
    }
  }
  // The wave's greatest listed logit into the block's, before a barrier; then what all came to.
  __device__ __forceinline__ void publish(const DistillParams& p, Shared& s) {
    float top = -kInf;
    each(p, [&](int e, int, float) { top = fmaxf(top, z(e)); });
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) s.z[threadIdx.x >> 6] = top;
  }
  // (the row's, in scalar registers: in vector ones they would not fit beside a held row)
  __device__ __forceinline__ void collect(const Shared& s) {
    t_max = uniform(waves_max<W>(s.t));
    z_max = uniform(waves_max<W>(s.z));
    n = __builtin_amdgcn_readfirstlane(waves_sum<W>(s.n));
  }
  // Sums of q (without lse: of its exponentials about the maximum), of
  // q (log q - (z - z_max) / T) and of the student's exponentials about z_max. Into the
  // block's sums with the thread's share of the rest, before a barrier; then from them.
  __device__ __forceinline__ void sums(const DistillParams& p, float rest, Shared& s) {
    q_sum = a_sum = 0.0;
    float zs = 0.0f;
    shift = p.lse ? static_cast<double>(lse) : static_cast<double>(t_max) * p.inv_t;
    const float base = z_max == -kInf ? 0.0f : z_max;
    each(p, [&](int e, int, float t) {
      const double log_q = static_cast<double>(t) * p.inv_t - shift, q = exp(log_q);
      q_sum += q;
      if (q != 0.0) a_sum += q * (log_q - (static_cast<double>(z(e)) - base) * p.inv_t);
      zs += exp_t(z(e) - base, p.c);
    });
    // (threads' sums meet in fp64: the loss is a small difference of logarithms, and
    // a rounding of the total by 2^-24 is 2e-6 of a loss of 0.03)
    const double r64 = wave_sum(static_cast<double>(rest)), z64 = wave_sum(static_cast<double>(zs));
    q_sum = wave_sum(q_sum);
    a_sum = wave_sum(a_sum);
    if ((threadIdx.x & 63) == 0) {
      s.rest[threadIdx.x >> 6] = r64;
      s.s[threadIdx.x >> 6] = z64;
      s.q[threadIdx.x >> 6] = q_sum;
      s.a[threadIdx.x >> 6] = a_sum;
    }
  }
  __device__ __forceinline__ void finish(const Shared& s) {
    q_sum = waves_sum<W>(s.q);
    a_sum = waves_sum<W>(s.a);
    z_sum = waves_sum<W>(s.s);
  }
};

// What a row comes to. The rest's exponentials are rest 2^base (base in powers of
// two: exp(u) = 2^(u log2 e)), the list's z_sum 2^(z_max c).
struct RowSums {
  double rest, base, top, total;  // total: of both, times 2^-top
  double above;                   // top, from z_max: of a list of masks no digit of 1e38 is left
  double q_rest, q_all, q_norm, p_rest, list_scale;
  template <int DT, int THREADS>
  __device__ __forceinline__ RowSums(const DistillParams& p, const List<DT, THREADS>& l, double rest_, double base_)
      : rest(rest_), base(base_) {
    const double c = static_cast<double>(p.c.hi) + p.c.lo;
    const double dz = l.z_max == -kInf ? base : l.z_max * c;
    top = rest > 0.0 ? fmax(base, dz) : dz;
    above = top - (l.z_max == -kInf ? 0.0 : dz);
    const double r = rest > 0.0 ? rest * exp2(base - top) : rest;  // (NaN stays)
    list_scale = exp2(dz - top);
    total = r + l.z_sum * list_scale;
    p_rest = r / total;
    // (where no unlisted logit is above minus infinity there is no such outcome)
    q_rest = 0.0;
    q_norm = 1.0;
    if (p.lse) q_rest = rest == 0.0 ? 0.0 : 1.0 - l.q_sum < 0.0 ? 0.0 : 1.0 - l.q_sum;
    else q_norm = 1.0 / l.q_sum;
    q_all = p.lse ? l.q_sum + q_rest : 1.0;
  }
  template <int DT, int THREADS>
  __device__ __forceinline__ float loss(const DistillParams& p, const List<DT, THREADS>& l) const {
    if (l.n < 0) return __builtin_nanf("");
    if (l.n == 0) return 0.0f;
    constexpr double ln2 = 0.69314718055994530942;
    const double log_total = log(total), log_p = log_total + above * ln2;
    double x = p.lse ? l.a_sum + l.q_sum * log_p : l.a_sum * q_norm - log(l.q_sum) + log_p;
    if (q_rest > 0.0) x += q_rest * (log(q_rest) - (log(rest) + (base - top) * ln2 - log_total));
    return static_cast<float>(x);
  }
  // The gradient on the rest is rest_gradient * (term of the rest's sum).
  __device__ __forceinline__ double rest_gradient(const DistillParams& p) const {
    return rest == 0.0 ? 0.0 : p.scale * p.inv_t * (q_all * p_rest - q_rest) / rest;
  }
  template <int DT, int THREADS>
  __device__ __forceinline__ void list_gradients(const DistillParams& p, const List<DT, THREADS>& l, uint8_t* dz) const {
    const double gs = p.scale * p.inv_t, f = list_scale / total * q_all;
    const float base_z = l.z_max == -kInf ? 0.0f : l.z_max;
    l.each(p, [&](int e, int id, float t) {
      const double q = exp(static_cast<double>(t) * p.inv_t - l.shift) * q_norm;
      store_elem<DT>(dz, id, static_cast<float>(gs * (static_cast<double>(exp_t(l.z(e) - base_z, p.c)) * f - q)));
    });
  }
};

// A barrier for what the block's threads have written to LDS; loads from memory
// stay in flight (__syncthreads waits for them).
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Piece i of a gradient row, laid out as piece_bytes reads it. The gradient passes by
// the caches: 2044 rows of 151936 286 us by plain stores and loads, 254 by these
// stores, 241 by such loads too of the pieces that are read once. Between the head's
// product and its backward, the gradient over the logits, such rows gain 2 % of the
// three (1247 us against 1269, 2048 rows and 896 columns of the head), rows that the
// last-level cache would hold lose as much (of 49152, 576 columns: 374 against 368).
template <int DT>
__device__ __forceinline__ void store_piece(uint8_t* row, int i, int V, uint4 o) {
  constexpr int E = kPiece<DT>, ES = 16 / E;
  if ((i + 1) * E <= V) {
    __builtin_nontemporal_store(u32x4u{o.x, o.y, o.z, o.w}, reinterpret_cast<u32x4u*>(row + static_cast<uint32_t>(i * 16)));
    return;
  }
  const uint32_t w[4] = {o.x, o.y, o.z, o.w};
  const int start = V >= E ? V - E : 0;
#pragma unroll
  for (int k = 0; k < E; ++k) {
    if (start + k < i * E || start + k >= V) continue;
    if constexpr (ES == 4) reinterpret_cast<uint32_t*>(row)[start + k] = w[k];
    else reinterpret_cast<uint16_t*>(row)[start + k] = static_cast<uint16_t>((k & 1) ? w[k >> 1] >> 16 : w[k >> 1]);
  }
}

// One workgroup per row, the row held in registers, LDS and, past both, in memory: N,
// M and R pieces of 16 bytes per thread. A bitmap of the listed
// ids in LDS takes them out of it (minus infinity), so the rest's sum is formed of
// its own terms: as the total less the listed it would have no digit left where
// the list has nearly all the mass. The listed logits are gathered by the threads
// that hold their list entries, whose gradients are written over the row's.
//
// With one row of 16-bit logits to a CU's registers nothing overlaps a row but
// itself, and 2 exponentials a logit (4 issue slots each) take as long as the
// row's loads. So the sum does not wait for the row's maximum: it runs about the
// maximum of the first pieces to arrive, piece by piece as the others do, and
// only a sum outside 2^-64 .. 2^64, or far from zero, is formed again about the
// maximum itself.
// exp(v / T) is 2^(v hi - b), one fused multiply-add: b is any number, and what
// hi lacks of log2(e) / T is made up in the sum's base, to first order, by the
// mean of v (over one in E of the terms). The gradient takes the same terms times
// one factor (in the exponent it would save that multiplication, and be off by
// 2^-24 of the largest logit).
//
// Two rows to a CU hide one another's waits: 2044 16-bit rows of 65536 logits took
// 181 us by one block of 1024 threads a CU and 121 by two of 512, and 1022 float32
// rows of 49152 108 and 88. So M further pieces of a thread lie in LDS, and R more,
// of rows past both, are read twice, for the sum through the registers of the held
// ones before these come and for the gradient as they leave: 2044 rows of 151936
// took 326 us by a CU a row, all held, and 305 so, although 14 of a thread's 37 pieces
// (38 % of the row) are read again. What else the two rows took from one another were
// their ways through the caches (store_piece): 242 us now, 5.1 TB/s of one reading and
// one writing, 6.1 with what is read again.
template <int DT, int THREADS, int N, int M, int R>
__global__ __launch_bounds__(THREADS, 4) void distill_held(DistillParams p) {
  constexpr int E = kPiece<DT>, ES = 16 / E, W = THREADS / 64;
  extern __shared__ uint32_t bitmap[];  // a bit per logit, a word more, and the list
  __shared__ typename List<DT, THREADS>::Shared s;
  __shared__ float s_first[W], s_ve[W], s_e[W];
  __shared__ float s_g;
  __shared__ uint4 beside[M ? M * THREADS : 1];  // pieces N .. N + M - 1
  static_assert(R <= N, "the pieces that are read again pass through the held ones' registers");
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t row = blockIdx.x;
  const int V = p.V, pieces = (V + E - 1) / E;
  const uint8_t* z = static_cast<const uint8_t*>(p.z) + row * p.ldz * ES;
  uint8_t* dz = static_cast<uint8_t*>(p.dz) + row * p.ldd * ES;

  List<DT, THREADS> l(bitmap + (V + 31) / 32 + 1, p.k);
  const typename List<DT, THREADS>::Entries entries = l.load(p, row);
  // (pieces past the end are the row's last 16 bytes, none of them its own)
  uint4 r[N];
  auto first = [&](int t, int j) __attribute__((always_inline)) { return min((j * THREADS + t) * E, V - E); };
  // (anew: a copy of the thread's index whose products no earlier pass has kept)
  auto anew = [&]() __attribute__((always_inline)) {
    int t = tid;
    asm volatile("" : "+v"(t));
    return t;
  };
  uint4 early[M ? M : 1];  // on their way to LDS
#pragma unroll
  for (int j = 0; j < M; ++j) early[j] = ld16nt(z + static_cast<uint32_t>(first(tid, N + j) * ES));
  constexpr int AHEAD = R > 8 ? 8 : N;
#pragma unroll
  for (int j = 0; j < AHEAD; ++j)
    r[j] = j < R ? ld16(z + static_cast<uint32_t>(first(tid, N + M + j) * ES)) : ld16nt(z + static_cast<uint32_t>(first(tid, j) * ES));
  for (int i = tid; i <= (V + 31) / 32; i += THREADS) bitmap[i] = 0;
  lds_barrier();
  l.mark(p, entries, z, bitmap, s);
#pragma unroll
  for (int j = AHEAD; j < N; ++j) {  // (the list's registers before these)
    int at = first(tid, j < R ? N + M + j : j) * ES;
    asm volatile("" : "+v"(at));
    r[j] = ld16(z + static_cast<uint32_t>(at));
  }
  {
    float v[E], mx = -kInf;
    widen<DT>(M ? early[0] : r[0], v);
#pragma unroll
    for (int k = 0; k < E; ++k) mx = fmaxf(mx, v[k]);
    mx = wave_max(mx);
    if (lane == 0) s_first[wave] = mx;
  }
  lds_barrier();
  // (the values are unpacked anew in each pass, not kept: fresh hides that they are the same)
  auto fresh = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < N; ++j) asm volatile("" : "+v"(r[j].x), "+v"(r[j].y), "+v"(r[j].z), "+v"(r[j].w));
  };
  // (A mask is no maximum: about itself its terms would be one where its product with log2(e) / T is exact. About
  // zero each is zero.)
  float about = uniform(waves_max<W>(s_first));
  if (about <= kMasked) about = 0.0f;
  float sum, ve, se;
  auto add_up = [&](auto takes) __attribute__((always_inline)) {
    if (!(__builtin_fabsf(about * p.c.hi) < kInf)) about = 0.0f;  // (so a sum past the floats becomes infinite)
    // (far from zero the first sum is only one to be formed again)
    constexpr bool again = !decltype(takes)::value;
    const ExpScale c = again ? scale_at<DT>(about, p.c) : p.c;
    const bool apart = again && DT == MR_F32 && is_far(about, p.c);
    const float b = -about * c.hi;
    auto term = [&](float v) __attribute__((always_inline)) {
      float x = __builtin_fmaf(v, c.hi, b);
      if (apart) {
        const float d = v - about;
        x = __builtin_fmaf(d, c.hi, d * c.lo);
      }
      return __builtin_amdgcn_exp2f(x);
    };
    const int t = anew();
    float s0 = 0.0f, s1 = 0.0f;
    ve = se = 0.0f;
    auto one = [&](int j, uint4& q, auto takes) __attribute__((always_inline)) {
      if constexpr (decltype(takes)::value) {
        const int at = first(t, j), drop = min((j * THREADS + t) * E - at, E);
        const uint32_t bits = __builtin_amdgcn_alignbit(bitmap[(at >> 5) + 1], bitmap[at >> 5], at & 31) | ((1u << drop) - 1);
        if (bits & ((1u << E) - 1)) take_out<DT>(q, bits);
      }
      float v[E];
      widen<DT>(q, v);
#pragma unroll
      for (int k = 0; k < E; k += 2) {
        const float e0 = term(v[k]);
        if (k == 0) {
          ve = __builtin_fmaf(fmaxf(v[0], -1e30f), e0, ve);
          se += e0;
        }
        s0 += e0;
        s1 += term(v[k + 1]);
      }
      // Here, as the pieces arrive: left alone the sums move behind the next barrier,
      // and the bitmap's words of every piece are read ahead (40 registers).
      // (And of float32 pieces, copies from before the listed were taken out are kept.)
      if constexpr (DT == MR_F32)
        asm volatile("" : "+v"(s0), "+v"(s1), "+v"(ve), "+v"(se), "+v"(q.x), "+v"(q.y), "+v"(q.z), "+v"(q.w));
      else
        asm volatile("" : "+v"(s0), "+v"(s1), "+v"(ve), "+v"(se));
      if (j & 1) __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int j = 0; j < M; ++j) {
      if constexpr (decltype(takes)::value) {
        one(N + j, early[j], takes);
        beside[j * THREADS + tid] = early[j];
      } else {
        uint4 q = beside[j * THREADS + tid];
        one(N + j, q, takes);
      }
    }
    if constexpr (decltype(takes)::value) {
#pragma unroll
      for (int j = 0; j < R; ++j) {
        one(N + M + j, r[j], takes);
        int at = first(t, j) * ES;
        asm volatile("" : "+v"(at));  // (behind the sum, whose piece's registers it takes)
        r[j] = ld16nt(z + static_cast<uint32_t>(at));
      }
    } else {
#pragma unroll 1
      for (int j = 0; j < R; ++j) {
        uint4 q = ld16(z + static_cast<uint32_t>(first(t, N + M + j) * ES));
        one(N + M + j, q, std::true_type{});
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) one(j, r[j], takes);
    sum = s0 + s1;
    ve = wave_sum(ve);
    se = wave_sum(se);
    if (lane == 0) {
      s_ve[wave] = ve;
      s_e[wave] = se;
    }
  };
  add_up(std::true_type{});
  l.publish(p, s);
  __syncthreads();
  l.collect(s);
  l.sums(p, sum, s);
  __syncthreads();  // (and every read of the row is done)
  const double rest0 = waves_sum<W>(s.rest);
  // (the row's values, one for all lanes: what a branch of a wave keeps of both sides spilled)
  const bool anew_about = !(rest0 > 0x1p-64 && rest0 < 0x1p64) || is_far(about, p.c);  // (or a NaN)
  if (__builtin_amdgcn_readfirstlane(anew_about)) {
    fresh();
    float mx = -kInf;
    auto most = [&](uint4 q) __attribute__((always_inline)) {
      float v[E];
      widen<DT>(q, v);
#pragma unroll
      for (int k = 0; k < E; ++k) mx = fmaxf(mx, v[k]);
    };
#pragma unroll
    for (int j = 0; j < N; ++j) most(r[j]);
#pragma unroll
    for (int j = 0; j < M; ++j) most(beside[j * THREADS + tid]);
#pragma unroll 1
    for (int j = 0; j < R; ++j) {
      const int at = first(tid, N + M + j), drop = min(((N + M + j) * THREADS + tid) * E - at, E);
      uint4 q = ld16(z + static_cast<uint32_t>(at * ES));
      const uint32_t bits = __builtin_amdgcn_alignbit(bitmap[(at >> 5) + 1], bitmap[at >> 5], at & 31) | ((1u << drop) - 1);
      take_out<DT>(q, bits);
      most(q);
    }
    mx = wave_max(mx);
    if (lane == 0) s_first[wave] = mx;
    __syncthreads();
    about = uniform(waves_max<W>(s_first));
    if (about <= kMasked) about = 0.0f;  // (every term is then zero)
    fresh();
    add_up(std::false_type{});
    const double r64 = wave_sum(static_cast<double>(sum));
    if (lane == 0) s.rest[wave] = r64;
    __syncthreads();
  }
  // What the row comes to, from the block's sums (a wave or all).
  auto row_sums = [&]() __attribute__((always_inline)) {
    const double lo = static_cast<double>(p.c.lo);
    const float v = uniform(waves_sum<W>(s_ve)), e = uniform(waves_sum<W>(s_e));
    l.finish(s);
    const double rest = waves_sum<W>(s.rest);
    // (a peak that the sampled terms lack is one or a few logits, whose terms are the sum)
    const float f = uniform(static_cast<float>(rest)), mean = mean_logit<E>(f, v, e, about + __builtin_amdgcn_logf(f) / p.c.hi);
    return RowSums(p, l, rest,
                   is_far(about, p.c) ? far_base(about, p.c)
                                      : static_cast<double>(about * p.c.hi) + lo * (rest > 0.0 ? static_cast<double>(mean) : about));
  };
  const bool none = l.n == 0;
  if (p.dz) {
    // (one wave works the factor out: in every wave its float64 registers would
    // not fit beside the row)
    if (wave == 0) {
      const RowSums x = row_sums();
      const double g = l.n < 0 ? __builtin_nan("") : x.rest_gradient(p);
      if (lane == 0)
        s_g = static_cast<float>(DT == MR_F32 ? g * exp2(about * (static_cast<double>(p.c.hi) + p.c.lo) - x.base) : g);
    }
    __syncthreads();
    const ExpScale c = scale_at<DT>(about, p.c);
    const float g = uniform(s_g), b = -about * c.hi;
    const int t = anew();
    fresh();
    auto put = [&](int j, uint4 q) __attribute__((always_inline)) {
      const int i = j * THREADS + t;
      if (i >= pieces) return;
      uint4 o = gradient_piece<DT>(q, about, b, g, c);
      if (none) o = make_uint4(0, 0, 0, 0);
      store_piece<DT>(dz, i, V, o);
      if (DT == MR_F32) __builtin_amdgcn_sched_barrier(0);  // (else pieces in float32 are worked on together, and spill)
    };
#pragma unroll
    for (int j = 0; j < N; ++j) {
      put(j, r[j]);
      if (j < R) r[j] = ld16nt(z + static_cast<uint32_t>(first(t, N + M + j) * ES));
    }
#pragma unroll
    for (int j = 0; j < M; ++j) put(N + j, beside[j * THREADS + tid]);
#pragma unroll
    for (int j = 0; j < R; ++j) put(N + M + j, r[j]);
    __syncthreads();  // the rest's stores are done where the list's follow
  }
  const RowSums x = row_sums();
  if (tid == 0) p.row_loss[row] = x.loss(p, l);
  if (p.dz && l.n > 0) x.list_gradients(p, l, dz);
}

// Rows whose gradient is not asked for, where they are longer than 2048 pieces, those
// too long to hold, which are read twice, and those shorter than a piece. Nothing is
// held, so a CU works on two rows by 1024 threads, on four by 512 and on eight by 256,
// which hide one another's waits: the loss alone of 2044 rows of 151936 bf16 logits 132,
// 115 and 108 us (5.7 TB/s), of 50304 80, 52 and 49; but 64 rows of 151936 23, 23 and 28.
// With the gradient the few rows at a time find more of themselves in the caches on
// the second reading: 2044 of 200000 374, 379 and 415.
template <int DT, int THREADS, bool GRAD>
__global__ __launch_bounds__(THREADS, 8) void distill_stream(DistillParams p) {
  constexpr int U = 4;
  constexpr int E = kPiece<DT>, ES = 16 / E, W = THREADS / 64;
  extern __shared__ uint32_t bitmap[];
  __shared__ typename List<DT, THREADS>::Shared s;
  __shared__ RunningSum::Shared<W> s_sum;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int V = p.V, pieces = (V + E - 1) / E;
  const uint8_t* z = static_cast<const uint8_t*>(p.z) + row * p.ldz * ES;
  uint8_t* dz = static_cast<uint8_t*>(p.dz) + row * p.ldd * ES;
  List<DT, THREADS> l(bitmap + (V + 31) / 32 + 1, p.k);
  const typename List<DT, THREADS>::Entries entries = l.load(p, row);
  for (int i = tid; i <= (V + 31) / 32; i += THREADS) bitmap[i] = 0;
  lds_barrier();
  l.mark(p, entries, z, bitmap, s);
  lds_barrier();
  auto get = [&](int i, auto last) __attribute__((always_inline)) {
    return V >= E ? piece_bytes<DT, decltype(last)::value>(z, i, V) : short_row<DT>(z, V);
  };
  // the listed elements of a piece and those that are not its own
  auto left_out = [&](int i) __attribute__((always_inline)) {
    if (V < E) return i ? 0xffu : bitmap[0] & 0xffu;
    const int at = min(i * E, V - E);
    return (__builtin_amdgcn_alignbit(bitmap[(at >> 5) + 1], bitmap[at >> 5], at & 31) | piece_drop<DT>(i, V)) & ((1u << E) - 1);
  };
  RunningSum running;
  for (int i0 = tid; i0 < pieces; i0 += U * THREADS) {
    uint4 q[U];
#pragma unroll
    for (int j = 0; j < U; ++j) q[j] = get(i0 + j * THREADS, std::bool_constant<!GRAD>{});
    float mx = -kInf;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (const uint32_t bits = left_out(i0 + j * THREADS)) take_out<DT>(q[j], bits);
      float v[E];
      widen<DT>(q[j], v);
#pragma unroll
      for (int k = 0; k < E; ++k) mx = fmaxf(mx, v[k]);
    }
    running.add<DT, U>(q, mx, p.c);
  }
  running.publish<W>(s_sum);
  l.publish(p, s);
  __syncthreads();
  l.collect(s);
  l.sums(p, 0.0f, s);
  __syncthreads();  // (and the list's reads of the row are done)
  l.finish(s);
  BlockSum<W, E> rest(s_sum, p.c);
  const float about = rest.max > kMasked ? rest.max : 0.0f;
  if (is_far(about, p.c)) {
    float sum = 0.0f;
    for (int i = tid; i < pieces; i += THREADS) {
      uint4 q = get(i, std::false_type{});
      take_out<DT>(q, left_out(i));
      float v[E];
      widen<DT>(q, v);
#pragma unroll
      for (int k = 0; k < E; ++k) sum += exp_t(v[k] - about, p.c);
    }
    const double r64 = wave_sum(static_cast<double>(sum));
    if ((tid & 63) == 0) s.rest[tid >> 6] = r64;
    __syncthreads();
    rest.sum = waves_sum<W>(s.rest);
    rest.exponent = far_base(about, p.c);
  }
  const RowSums x(p, l, rest.sum, rest.exponent);
  if (tid == 0) p.row_loss[row] = x.loss(p, l);
  if constexpr (!GRAD) return;
  const bool none = l.n == 0;
  const double g64 = l.n < 0 ? __builtin_nan("") : x.rest_gradient(p);
  const ExpScale c = scale_at<DT>(about, p.c);
  const float base = -about * c.hi;
  const float g = static_cast<float>(DT == MR_F32 ? g64 * exp2(about * (static_cast<double>(p.c.hi) + p.c.lo) - x.base) : g64);
  for (int i0 = tid; i0 < pieces; i0 += U * THREADS) {
    uint4 q[U];
#pragma unroll
    for (int j = 0; j < U; ++j) q[j] = get(i0 + j * THREADS, std::true_type{});
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = i0 + j * THREADS;
      if (i >= pieces) continue;
      if (const uint32_t bits = left_out(i)) take_out<DT>(q[j], bits);
      uint4 o = gradient_piece<DT>(q[j], about, base, g, c);
      if (none) o = make_uint4(0, 0, 0, 0);
      store_piece<DT>(dz, i, V, o);
    }
  }
  __syncthreads();  // the rest's stores are done where the list's follow
  if (l.n > 0) x.list_gradients(p, l, dz);
}

// loss = scale * sum of the row losses, in a fixed order (fp64 partials).
__global__ __launch_bounds__(1024) void sum_rows(const float* __restrict__ row_loss, int64_t T, float scale,
                                                 float* __restrict__ loss_out) {
  __shared__ double sm[16];
  double acc = 0.0;
  for (int64_t i = threadIdx.x; i < T; i += 1024) acc += static_cast<double>(row_loss[i]);
  acc = wave_sum(acc);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < 16; ++w) t += sm[w];
    loss_out[0] = static_cast<float>(t * static_cast<double>(scale));
  }
}

bool element_aligned(const void* p, int es) { return reinterpret_cast<uintptr_t>(p) % es == 0; }

}  // namespace
}  // namespace mr

extern "C" {

int mr_top_logits(const void* logits, int dtype, int64_t ld, int64_t T, int64_t V, int k, double temperature,
                  float* values, int32_t* ids, float* lse, void* stream) {
  using namespace mr;
  clear_error();
  if (T < 0 || V <= 0) return fail(MR_EINVAL, "mr_top_logits: bad sizes T=%lld V=%lld", static_cast<long long>(T),
                                   static_cast<long long>(V));
  if (!valid_dtype(dtype)) return fail(MR_EINVAL, "mr_top_logits: bad dtype %d", dtype);
  if (k < 1 || k > kMaxTop || k > V)
    return fail(MR_EINVAL, "mr_top_logits: k=%d must lie in [1, %d] and not pass V", k, kMaxTop);
  if (!(temperature >= kMinTemperature && temperature <= kMaxTemperature))
    return fail(MR_EINVAL, "mr_top_logits: the temperature must lie in [1/1024, 1024]");
  if (T == 0) return MR_OK;
  if (!logits || !values || !ids) return fail(MR_EINVAL, "mr_top_logits: null pointer");
  if (ld < V) return fail(MR_EINVAL, "mr_top_logits: the leading dimension is smaller than V");
  if (T > 0x7fffffff || V > 0x7fffffff) return fail(MR_EINVAL, "mr_top_logits: too large");
  const int es = dtype_bytes(dtype);
  if (!element_aligned(logits, es) || !element_aligned(values, 4) || !element_aligned(ids, 4) || !element_aligned(lse, 4))
    return fail(MR_EINVAL, "mr_top_logits: a pointer is not aligned to its elements");
  {
    const int64_t nx = ((T - 1) * ld + V) * es, no = T * k * 4;
    if (overlap(values, no, logits, nx) || overlap(ids, no, logits, nx) || overlap(values, no, ids, no) ||
        (lse && (overlap(lse, T * 4, logits, nx) || overlap(lse, T * 4, values, no) || overlap(lse, T * 4, ids, no))))
      return fail(MR_EINVAL, "mr_top_logits: the outputs must not overlap the logits or each other");
  }
  TopParams p{logits, ld, V, k, exp_scale(temperature), temperature, values, ids, lse};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 g(static_cast<unsigned>(T));
  // Short rows by blocks of 256 threads, eight to a CU, longer ones by four of 512,
  // where these have maxima enough for lists of k: 2044 rows of 20000 bf16 logits 67 us
  // by 1024 threads, 38 by 512, 32 by 256; of 50304 78, 51, 57; of 151936 144, 138, 163.
  const int threads = V <= 24576 && k <= 256 ? 256 : k <= 512 ? 512 : 1024;
  if (too_many_blocks(T, threads)) return fail(MR_EINVAL, "mr_top_logits: too large, a launch takes %lld such rows",
                                               0xffffffffll / threads);
#define MR_TOP(DT)                                                                                          \
  do {                                                                                                      \
    if (threads == 256) hipLaunchKernelGGL((top_rows<DT, 256>), g, dim3(256), 0, s, p);                      \
    else if (threads == 512) hipLaunchKernelGGL((top_rows<DT, 512>), g, dim3(512), 0, s, p);                 \
    else hipLaunchKernelGGL((top_rows<DT, 1024>), g, dim3(1024), 0, s, p);                                   \
  } while (0)
  if (dtype == MR_BF16) MR_TOP(MR_BF16);
  else if (dtype == MR_F16) MR_TOP(MR_F16);
  else MR_TOP(MR_F32);
#undef MR_TOP
  MR_LAUNCH_CHECK("mr_top_logits");
  return MR_OK;
}

int mr_distill(const void* logits, int dtype, int64_t ld, int64_t T, int64_t V, const float* top_values,
               const int32_t* top_ids, int k, const float* top_lse, double temperature, float scale, float* row_loss,
               float* loss_out, void* dlogits, int64_t ldd, void* stream) {
  using namespace mr;
  clear_error();
  if (T < 0 || V <= 0) return fail(MR_EINVAL, "mr_distill: bad sizes T=%lld V=%lld", static_cast<long long>(T),
                                   static_cast<long long>(V));
  if (V > kBitmapMaxV) return fail(MR_EINVAL, "mr_distill: vocabularies of more than %d", kBitmapMaxV);
  if (!valid_dtype(dtype)) return fail(MR_EINVAL, "mr_distill: bad dtype %d", dtype);
  if (k < 1 || k > kMaxTop) return fail(MR_EINVAL, "mr_distill: k=%d must lie in [1, %d]", k, kMaxTop);
  if (!(temperature >= kMinTemperature && temperature <= kMaxTemperature))
    return fail(MR_EINVAL, "mr_distill: the temperature must lie in [1/1024, 1024]");
  if (T > 0 && (!row_loss || !logits || !top_values || !top_ids)) return fail(MR_EINVAL, "mr_distill: null pointer");
  if (ld < V || (dlogits && ldd < V)) return fail(MR_EINVAL, "mr_distill: a leading dimension is smaller than V");
  if (T > 0x7fffffff) return fail(MR_EINVAL, "mr_distill: too many rows");
  const int es = dtype_bytes(dtype);
  if (!element_aligned(logits, es) || !element_aligned(dlogits, es) || !element_aligned(top_values, 4) ||
      !element_aligned(top_ids, 4) || !element_aligned(top_lse, 4) || !element_aligned(row_loss, 4) ||
      !element_aligned(loss_out, 4))
    return fail(MR_EINVAL, "mr_distill: a pointer is not aligned to its elements");
  if (T > 0) {
    // The gradient may be written over the logits (the same rows), else the
    // outputs share nothing with what is read or each other.
    const int64_t nz = ((T - 1) * ld + V) * es, nd = ((T - 1) * ldd + V) * es, nl = T * k * 4;
    const void* reads[4] = {logits, top_values, top_ids, top_lse};
    const int64_t nr[4] = {nz, nl, nl, T * 4};
    const void* writes[3] = {dlogits, row_loss, loss_out};
    const int64_t nw[3] = {nd, T * 4, 4};
    for (int a = 0; a < 3; ++a) {
      if (!writes[a]) continue;
      for (int b = 0; b < 4; ++b) {
        if (!reads[b] || (a == 0 && b == 0 && dlogits == logits && ldd == ld)) continue;
        if (overlap(writes[a], nw[a], reads[b], nr[b]))
          return fail(MR_EINVAL, "mr_distill: an output overlaps an input (the gradient may only be the logits themselves)");
      }
      for (int b = a + 1; b < 3; ++b)
        if (writes[b] && overlap(writes[a], nw[a], writes[b], nw[b]))
          return fail(MR_EINVAL, "mr_distill: the outputs overlap");
    }
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (T > 0) {
    DistillParams p{logits, ld, static_cast<int>(V), k, top_values, top_ids, top_lse, exp_scale(temperature),
                    1.0 / temperature, scale, row_loss, dlogits, ldd};
    const dim3 g(static_cast<unsigned>(T));
    const size_t lds = static_cast<size_t>((V + 31) / 32 + 1) * 4 + static_cast<size_t>(k) * 8;
    const int64_t pieces = (V * es + 15) / 16;
    // what 7 pieces a thread and the block's sums leave of half a CU's LDS
    constexpr size_t kTwoRows = 81920 - 512 * 7 * 16 - 2048;
#define MR_ROWS(KERNEL, THREADS)                                                                              \
  do {                                                                                                       \
    if (too_many_blocks(T, THREADS))                                                                         \
      return fail(MR_EINVAL, "mr_distill: too many rows, a launch takes %lld", 0xffffffffll / (THREADS));     \
    hipLaunchKernelGGL(KERNEL, g, dim3(THREADS), lds, s, p);                                                  \
  } while (0)
#define MR_DISTILL(DT, THREADS, N, M, R) MR_ROWS((distill_held<DT, THREADS, N, M, R>), THREADS)
    // The fewest threads that hold the row in at most 8 pieces each, then more pieces,
    // some of them in LDS, then some read twice, as long as two rows fit a CU;
    // the loss alone by small blocks where there are rows for eight of them a CU and
    // room for their bitmaps; a row that is read twice by the whole of half a CU
#define MR_STREAM(DT, THREADS, GRAD) MR_ROWS((distill_stream<DT, THREADS, GRAD>), THREADS)
#define MR_DISTILL_D(DT)                                                                                 \
  do {                                                                                                   \
    if (V * es < 16 || (!dlogits && pieces > 256 * 8)) {                                                   \
      if (dlogits) MR_STREAM(DT, 1024, true);                                                              \
      else if (T >= 1024 && lds <= 20480) MR_STREAM(DT, 256, false);                                       \
      else if (lds <= 40960) MR_STREAM(DT, 512, false);                                                    \
      else MR_STREAM(DT, 1024, false);                                                                     \
    } else if (pieces <= 256 * 4) MR_DISTILL(DT, 256, 4, 0, 0);                                               \
    else if (pieces <= 256 * 8) MR_DISTILL(DT, 256, 8, 0, 0);                                               \
    else if (pieces <= 512 * 8) MR_DISTILL(DT, 512, 8, 0, 0);                                               \
    else if (pieces <= 512 * 16) MR_DISTILL(DT, 512, 16, 0, 0);                                             \
    else if (pieces <= 512 * 20) MR_DISTILL(DT, 512, 20, 0, 0);                                             \
    else if (pieces <= 512 * 24) MR_DISTILL(DT, 512, 17, 7, 0);                                             \
    else if (pieces <= 512 * 31) MR_DISTILL(DT, 512, 17, 6, 8);                                          \
    else if (pieces <= 512 * 39 && lds <= kTwoRows) MR_DISTILL(DT, 512, 16, 7, 16);                      \
    else if (pieces <= 512 * 40) MR_DISTILL(DT, 512, 17, 6, 17);                                           \
    else MR_STREAM(DT, 1024, true);                             \
  } while (0)
    if (dtype == MR_BF16) MR_DISTILL_D(MR_BF16);
    else if (dtype == MR_F16) MR_DISTILL_D(MR_F16);
    else MR_DISTILL_D(MR_F32);
#undef MR_DISTILL_D
#undef MR_STREAM
#undef MR_DISTILL
#undef MR_ROWS
    MR_LAUNCH_CHECK("mr_distill");
  }
  if (loss_out) {
    hipLaunchKernelGGL(sum_rows, dim3(1), dim3(1024), 0, s, row_loss, T, scale, loss_out);
    MR_LAUNCH_CHECK("mr_distill");
  }
  return MR_OK;
}

}  // extern "C"
