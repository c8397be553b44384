// Rotary positions of any layout for gfx950: halves or neighbours paired, the
// whole head or its first part, any position per token, frequencies of any
// scaling.
//
// For pair i of a head at position p, theta = p f_i and
//   (a, b) -> s (a cos theta - b sin theta, a sin theta + b cos theta),
// with (a, b) = (x_i, x_{i + r/2}) or (x_2i, x_{2i+1}) of the first r elements
// of the head; the backward is the transposed rotation, theta negated.
//
// An angle at a far position has lost its turn in float32 (position 10^6 at
// f = 1 is off by 0.03), so p f_i / 2 pi is formed in float64 and only its
// distance from the nearest whole number is narrowed: 2^-25 turns at most, plus
// 2^-53 of the product. A token's angles serve all its heads, so a block takes
// a few tokens, one thread computes one angle into LDS, and the heads read it
// there: no table of positions is read or kept, at any length.
//
// Bound by memory: an element is read and written once. 16384 tokens of 32 bf16
// heads of 128 take 50 us (268 MB, 5.4 TB/s), 4000 of 16 float16 heads, 32 of 64
// elements rotated, 6 us, and 8 tokens 3 us, where a call's own 8 us on the host are
// what counts. A thread has 4 x 32 bytes on their way while the angles are worked out.
//
// Loads and stores pass by the caches where another buffer receives whole heads whose
// halves are whole cache lines (of 128 bytes): that call takes 50 us so and 58 through
// the caches, of 65536 tokens 189 and 206. Elsewhere they do not. In place the product
// that wrote the rows has left them there and attention reads them next: product,
// rotation and attention of 16384 tokens of 16 + 2 heads of 128 (rows of 2560) took 325
// us past the caches, and take 320; of neighbours 334 and 321; of 14 + 2 heads of 64 half
// rotated 146 and 138. And neighbours or a head's rest, 32 bytes a thread, or halves
// under a line are parts of lines, which the caches put together: 65536 tokens of
// neighbours 302 us past them and 203 through them, of heads of 128 half rotated 275 and 213.
#include "mr_common.h"

namespace mr {
namespace {

constexpr int kRopeBlock = 256;
constexpr int kRopeUnits = 4;  // units of 16 + 16 bytes a thread has in flight

// A unit is 16 bytes of a's and 16 of b's (halves), or 32 consecutive bytes.
struct Unit {
  uint4 a, b;
};

struct RopeParams {
  const void* x;
  void* out;
  int64_t ldx, ldo;
  const int32_t* positions;
  const double* freq;
  int T, n_heads, d, pairs;  // pairs: r / 2
  float scale;
  int end;          // elements of a head that are visited: the rotated ones in place, else all
  int tokens;       // per block
  int head_units;   // units of a head, rotated ones first
  int rot_units;
};

__device__ __forceinline__ uint4 ld16(const uint8_t* p) {
  uint4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
__device__ __forceinline__ void st16(uint8_t* p, uint4 v) { __builtin_memcpy(p, &v, 16); }

// The same of 16-byte places, past the caches.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint4 ld16s(const uint8_t* p) {
  const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
  return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void st16s(uint8_t* p, uint4 v) {
  __builtin_nontemporal_store(u32x4{v.x, v.y, v.z, v.w}, reinterpret_cast<u32x4*>(p));
}

// E consecutive elements of a 16-byte register, widened, and back.
template <int DT, int E>
__device__ __forceinline__ void widen(uint4 r, float (&v)[E]) {
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
template <int DT, int E>
__device__ __forceinline__ uint4 narrow(const float (&v)[E]) {
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (DT == MR_F32) w[k] = __float_as_uint(v[k]);
    else if constexpr (DT == MR_BF16) w[k] = pack_bf16x2(v[2 * k], v[2 * k + 1]);
    else w[k] = static_cast<uint32_t>(f32_to_f16(v[2 * k])) | (static_cast<uint32_t>(f32_to_f16(v[2 * k + 1])) << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// VEC: every rotated unit is whole and every unit starts on 16 bytes; PAST: and what
// is moved passes by the caches.
template <int DT, bool HALF, bool BWD, bool VEC, bool PAST>
__global__ __launch_bounds__(kRopeBlock) void rope_any(RopeParams p) {
  constexpr int ES = DT == MR_F32 ? 4 : 2;  // bytes of an element
  constexpr int E = 16 / ES;                // pairs of a unit
  extern __shared__ float2 cs[];            // [tokens][pairs]: s cos, s sin
  const int t0 = static_cast<int>(blockIdx.x) * p.tokens;
  const int nt = min(p.tokens, p.T - t0);
  const uint32_t per_token = static_cast<uint32_t>(p.n_heads) * p.head_units;
  const uint32_t total = per_token * nt;
  const uint8_t* xb = static_cast<const uint8_t*>(p.x) + static_cast<int64_t>(t0) * p.ldx * ES;
  uint8_t* ob = static_cast<uint8_t*>(p.out) + static_cast<int64_t>(t0) * p.ldo * ES;

  // Where unit `idx` lies: its token, its first pair (rotated units) and the
  // element offsets of its two 16-byte pieces in the head row. n: elements of
  // each piece that belong to the unit (E unless it is the last of its kind).
  struct At {
    int tok, pair, a, b, na, nb;
    bool rot;
  };
  auto at = [&](uint32_t idx) __attribute__((always_inline)) {
    At u;
    u.tok = static_cast<int>(idx / per_token);
    const uint32_t rem = idx - u.tok * per_token;
    const int head = static_cast<int>(rem / p.head_units);
    const int k = static_cast<int>(rem) - head * p.head_units;
    const int h0 = head * p.d;
    u.rot = k < p.rot_units;
    u.pair = k * E;
    if (HALF && u.rot) {
      u.a = h0 + k * E;
      u.b = u.a + p.pairs;
      u.na = u.nb = VEC ? E : min(E, p.pairs - k * E);
    } else {
      // neighbours, or the unrotated rest: 2 E consecutive elements
      const int first = HALF ? 2 * p.pairs + (k - p.rot_units) * 2 * E : k * 2 * E;
      const int left = p.end - first;
      u.a = h0 + first;
      u.b = u.a + E;
      u.na = min(E, left);
      u.nb = max(0, min(E, left - E));
    }
    return u;
  };
  auto load = [&](const At& u) __attribute__((always_inline)) {
    const uint8_t* row = xb + static_cast<int64_t>(u.tok) * p.ldx * ES;
    Unit v{};
    if (PAST && u.na == E && u.nb == E) {
      v.a = ld16s(row + u.a * ES);
      v.b = ld16s(row + u.b * ES);
    } else if (u.na == E && u.nb == E) {
      v.a = ld16(row + u.a * ES);
      v.b = ld16(row + u.b * ES);
    } else {
      uint8_t buf[32] = {};
#pragma unroll
      for (int k = 0; k < E; ++k) {
        if (k < u.na) __builtin_memcpy(buf + k * ES, row + (u.a + k) * ES, ES);
        if (k < u.nb) __builtin_memcpy(buf + 16 + k * ES, row + (u.b + k) * ES, ES);
      }
      __builtin_memcpy(&v.a, buf, 16);
      __builtin_memcpy(&v.b, buf + 16, 16);
    }
    return v;
  };
  auto store = [&](const At& u, const Unit& v) __attribute__((always_inline)) {
    uint8_t* row = ob + static_cast<int64_t>(u.tok) * p.ldo * ES;
    if (PAST && u.na == E && u.nb == E) {
      st16s(row + u.a * ES, v.a);
      st16s(row + u.b * ES, v.b);
    } else if (u.na == E && u.nb == E) {
      st16(row + u.a * ES, v.a);
      st16(row + u.b * ES, v.b);
    } else {
      uint8_t buf[32];
      __builtin_memcpy(buf, &v.a, 16);
      __builtin_memcpy(buf + 16, &v.b, 16);
#pragma unroll
      for (int k = 0; k < E; ++k) {
        if (k < u.na) __builtin_memcpy(row + (u.a + k) * ES, buf + k * ES, ES);
        if (k < u.nb) __builtin_memcpy(row + (u.b + k) * ES, buf + 16 + k * ES, ES);
      }
    }
  };

  auto angles = [&]() __attribute__((always_inline)) {
    for (int i = threadIdx.x; i < nt * p.pairs; i += kRopeBlock) {
      const int tok = i / p.pairs, k = i - tok * p.pairs;
      const double turns = static_cast<double>(p.positions[t0 + tok]) * (p.freq[k] * 0.15915494309189535);
      const float part = static_cast<float>(turns - rint(turns));
      float sn, c;
      sincospif(2.0f * part, &sn, &c);
      cs[i] = make_float2(p.scale * c, (BWD ? -p.scale : p.scale) * sn);
    }
  };

  bool first = true;
  for (uint32_t base = threadIdx.x; first || base < total; base += kRopeBlock * kRopeUnits) {
    Unit v[kRopeUnits];
#pragma unroll
    for (int j = 0; j < kRopeUnits; ++j)
      if (base + j * kRopeBlock < total) v[j] = load(at(base + j * kRopeBlock));
    if (first) {  // (every thread, with its first loads in flight)
      angles();
      __syncthreads();
      first = false;
    }
#pragma unroll
    for (int j = 0; j < kRopeUnits; ++j) {
      if (base + j * kRopeBlock >= total) break;
      const At u = at(base + j * kRopeBlock);
      if (u.rot) {
        float a[E], b[E];
        widen<DT, E>(v[j].a, a);
        widen<DT, E>(v[j].b, b);
        const float2* c = cs + u.tok * p.pairs + u.pair;
        if constexpr (HALF) {
#pragma unroll
          for (int k = 0; k < E; ++k) {
            if (!VEC && k >= u.na) break;
            const float2 w = c[k];
            const float ya = a[k] * w.x - b[k] * w.y, yb = a[k] * w.y + b[k] * w.x;
            a[k] = ya;
            b[k] = yb;
          }
        } else {
#pragma unroll
          for (int k = 0; k < E; ++k) {
            if (!VEC && u.pair + k >= p.pairs) break;  // the unrotated rest of a unit
            const float2 w = c[k];
            float& xa = k < E / 2 ? a[2 * k] : b[2 * k - E];
            float& xb2 = k < E / 2 ? a[2 * k + 1] : b[2 * k + 1 - E];
            const float ya = xa * w.x - xb2 * w.y, yb = xa * w.y + xb2 * w.x;
            xa = ya;
            xb2 = yb;
          }
        }
        v[j].a = narrow<DT, E>(a);
        v[j].b = narrow<DT, E>(b);
      }
      store(u, v[j]);
    }
  }
}

}  // namespace
}  // namespace mr

extern "C" {

int mr_rope_positions(const void* x, int dtype, int64_t ldx, int64_t T, int n_heads, int head_dim,
                      const int32_t* positions, const double* frequencies, int rotary_dim, int pairing, float scale,
                      int backward, void* out, int64_t ldo, void* stream) {
  using namespace mr;
  clear_error();
  if (T < 0 || n_heads < 0 || head_dim <= 0)
    return fail(MR_EINVAL, "mr_rope_positions: bad sizes T=%lld n_heads=%d head_dim=%d", static_cast<long long>(T),
                n_heads, head_dim);
  if (!valid_dtype(dtype)) return fail(MR_EINVAL, "mr_rope_positions: bad dtype %d", dtype);
  if (pairing != MR_ROPE_HALF && pairing != MR_ROPE_INTERLEAVED)
    return fail(MR_EINVAL, "mr_rope_positions: unknown pairing %d", pairing);
  if (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > head_dim)
    return fail(MR_EINVAL, "mr_rope_positions: the rotated part %d must be even and at most the head's %d", rotary_dim,
                head_dim);
  if (T == 0 || n_heads == 0) return MR_OK;
  if (!x || !positions || !frequencies || !out) return fail(MR_EINVAL, "mr_rope_positions: null pointer");
  const int64_t width = static_cast<int64_t>(n_heads) * head_dim;
  if (width > (1 << 24) || head_dim > 4096)
    return fail(MR_EINVAL, "mr_rope_positions: heads of more than 4096 or rows of more than %d elements", 1 << 24);
  if (ldx < width || ldo < width) return fail(MR_EINVAL, "mr_rope_positions: a leading dimension is smaller than the heads");
  if (T > 0x7fffffff) return fail(MR_EINVAL, "mr_rope_positions: too many rows");
  const int es = dtype_bytes(dtype);
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) % es ||
      reinterpret_cast<uintptr_t>(positions) % 4 || reinterpret_cast<uintptr_t>(frequencies) % 8)
    return fail(MR_EINVAL, "mr_rope_positions: a pointer is not aligned to its elements");
  const bool in_place = x == out && ldx == ldo;
  const int64_t nx = ((T - 1) * ldx + width) * es, no = ((T - 1) * ldo + width) * es;
  if ((!in_place && overlap(x, nx, out, no)) || overlap(out, no, positions, T * 4) ||
      overlap(out, no, frequencies, rotary_dim * 4))
    return fail(MR_EINVAL, "mr_rope_positions: out must be x itself or share no memory with what is read");
  const int e = 16 / es;
  RopeParams p{};
  p.x = x;
  p.out = out;
  p.ldx = ldx;
  p.ldo = ldo;
  p.positions = positions;
  p.freq = frequencies;
  p.T = static_cast<int>(T);
  p.n_heads = n_heads;
  p.d = head_dim;
  p.pairs = rotary_dim / 2;
  p.scale = scale;
  const int visited = in_place ? rotary_dim : head_dim;
  p.end = visited;
  const bool half = pairing == MR_ROPE_HALF;
  p.rot_units = (p.pairs + e - 1) / e;
  p.head_units = p.rot_units + (visited - rotary_dim + 2 * e - 1) / (2 * e);
  if (!half) {
    p.rot_units = (rotary_dim + 2 * e - 1) / (2 * e);
    p.head_units = (visited + 2 * e - 1) / (2 * e);
  }
  // whole rotated units, and pieces of 16 bytes on 16-byte addresses
  const bool vec = p.pairs % e == 0 && head_dim % e == 0 && (ldx * es) % 16 == 0 && (ldo * es) % 16 == 0 &&
                   aligned16(x) && aligned16(out);
  const bool past = vec && half && !in_place && rotary_dim == head_dim && p.pairs * es % 128 == 0;
  // Tokens of a block: an angle for each of its threads, but blocks enough to
  // give every CU four, and 32 KB of angles at most.
  int64_t tokens = (kRopeBlock + p.pairs - 1) / p.pairs;
  const int64_t even = T / 1024;
  if (tokens > even) tokens = even > 0 ? even : 1;
  p.tokens = static_cast<int>(tokens);
  if (too_many_blocks((T + tokens - 1) / tokens, kRopeBlock))
    return fail(MR_EINVAL, "mr_rope_positions: too many rows, a launch takes %lld", 0xffffffffll / kRopeBlock * tokens);
  const dim3 grid(static_cast<unsigned>((T + tokens - 1) / tokens)), block(kRopeBlock);
  const size_t lds = static_cast<size_t>(tokens) * p.pairs * sizeof(float2);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define MR_ROPE(DT, HALF, BWD, VEC, PAST) hipLaunchKernelGGL((rope_any<DT, HALF, BWD, VEC, PAST>), grid, block, lds, s, p)
#define MR_ROPE_V(DT, HALF, BWD)                              \
  do {                                                        \
    if (HALF && past) MR_ROPE(DT, HALF, BWD, true, HALF);     \
    else if (vec) MR_ROPE(DT, HALF, BWD, true, false);        \
    else MR_ROPE(DT, HALF, BWD, false, false);                \
  } while (0)
#define MR_ROPE_D(DT)                                                                   \
  do {                                                                                  \
    if (half) { if (backward) MR_ROPE_V(DT, true, true); else MR_ROPE_V(DT, true, false); } \
    else { if (backward) MR_ROPE_V(DT, false, true); else MR_ROPE_V(DT, false, false); }    \
  } while (0)
  if (dtype == MR_BF16) MR_ROPE_D(MR_BF16);
  else if (dtype == MR_F16) MR_ROPE_D(MR_F16);
  else MR_ROPE_D(MR_F32);
#undef MR_ROPE_D
#undef MR_ROPE_V
#undef MR_ROPE
  MR_LAUNCH_CHECK("mr_rope_positions");
  return MR_OK;
}

}  // extern "C"
