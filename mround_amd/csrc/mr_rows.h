// Pieces of a row, as loaded and as floats, and sums over a wave: for kernels
// that hold rows in registers.
#pragma once

#include "mr_common.h"

namespace mr {

// V consecutive elements of type DT as they lie in memory: 8 on addresses of 16
// bytes, or one. Held raw between their load and their use, so that a row can
// be in flight while the one before it is worked on.
template <int DT, int V>
struct Piece {
  static constexpr int WORDS = V == 8 ? (DT == MR_F32 ? 8 : 4) : 1;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    if constexpr (V == 1) {
      if constexpr (DT == MR_F32) w[0] = static_cast<const uint32_t*>(p)[i];
      else w[0] = static_cast<const uint16_t*>(p)[i];
    } else {
      const char* a = static_cast<const char*>(p) + i * (DT == MR_F32 ? 4 : 2);
#pragma unroll
      for (int q = 0; q < WORDS / 4; ++q) {
        const u32x4_t r = reinterpret_cast<const u32x4_t*>(a)[q];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[4 * q + k] = r[k];
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int k = 0; k < WORDS; ++k) w[k] = 0;
  }
  // Its floats are to be made again from here on, not kept.
  __device__ __forceinline__ void hide() {
#pragma unroll
    for (int k = 0; k < WORDS; ++k) asm volatile("" : "+v"(w[k]));
  }
  __device__ __forceinline__ float get(int k) const {
    if constexpr (DT == MR_F32) return __uint_as_float(w[k]);
    const uint32_t x = V == 1 ? w[0] : w[k >> 1] >> (16 * (k & 1));
    if constexpr (DT == MR_BF16) return __uint_as_float(x << 16);
    return f16_to_f32(static_cast<uint16_t>(x));
  }
};

// V floats to V elements of type DT at index i, rounded once; NT passes by the caches.
template <int DT, int V, bool NT>
__device__ __forceinline__ void store_piece(void* p, int64_t i, const float (&x)[V]) {
  if constexpr (V == 1) {
    store_elem<DT>(p, i, x[0]);
  } else {
    uint32_t w[DT == MR_F32 ? 8 : 4];
    if constexpr (DT == MR_F32) {
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = __float_as_uint(x[k]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (DT == MR_BF16) {
          w[k] = pack_bf16x2(x[2 * k], x[2 * k + 1]);
        } else {  // (the float32 values themselves, as in store8)
          float lo = x[2 * k], hi = x[2 * k + 1];
          asm("" : "+v"(lo), "+v"(hi));
          w[k] = static_cast<uint32_t>(f32_to_f16(lo)) | (static_cast<uint32_t>(f32_to_f16(hi)) << 16);
        }
      }
    }
    char* a = static_cast<char*>(p) + i * (DT == MR_F32 ? 4 : 2);
#pragma unroll
    for (int q = 0; q < (DT == MR_F32 ? 2 : 1); ++q) {
      const u32x4_t r = {w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]};
      if constexpr (NT) __builtin_nontemporal_store(r, reinterpret_cast<u32x4_t*>(a) + q);
      else reinterpret_cast<u32x4_t*>(a)[q] = r;
    }
  }
}

// x of the lane that DPP control CTRL names (every lane active).
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x) { return __uint_as_float(dpp<CTRL>(__float_as_uint(x))); }
// Steps that meet all 16 lanes of a row: neighbours, pairs, halves mirrored, the row mirrored.
constexpr int kDppXor1 = 0xb1, kDppXor2 = 0x4e, kDppHalfMirror = 0x141, kDppMirror = 0x140;

__device__ __forceinline__ float row16_sum(float x) {
  x += dpp<kDppXor1>(x);
  x += dpp<kDppXor2>(x);
  x += dpp<kDppHalfMirror>(x);
  return x + dpp<kDppMirror>(x);
}

// The wave's sum, in every lane and the same bits in each.
__device__ __forceinline__ float wave_sum(float x) {
  const int r = __float_as_int(row16_sum(x));
  auto of = [&](int lane) { return __int_as_float(__builtin_amdgcn_readlane(r, lane)); };
  return (of(0) + of(16)) + (of(32) + of(48));
}

// The sum of x over the lanes up to each one (row by row of 16 lanes, then across them).
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // 1, 2, 4, 8 lanes down a row
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // the last of rows 0 and 2 to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // the last of row 1 to rows 2 and 3
  return x;
}

}  // namespace mr
