// Products grouped by expert: the rows of A, in the experts' order, times their
// expert's weight, and the weights' gradients over each expert's rows.
//
//   nt  C[r] = A[r] B[e]^T   (A's rows may lie at an index)      forward
//   nn  C[r] = A[r] B[e]                                         input gradients
//   tn  C[e] = A[rows of e]^T B[rows of e]                       weight gradients
//
// for the rows offsets[e] <= r < offsets[e + 1] of expert e, whose counts are on
// the device alone. The tiles, pipelines and epilogues are the ungrouped products'
// (mr_gemm_tiles.h); a block finds its expert and tile by itself.
#include "mr_gemm_tiles.h"

namespace mr {
namespace {

struct Grouped {
  int64_t M, N, K;  // (M or, with MN-major A, K: all experts' rows)
  const void* A;
  int64_t lda;
  const int32_t* index;
  int64_t a_rows;
  const void* B;
  int64_t ldb, b_step;
  const int32_t* offsets;
  int64_t experts;
  void* C;
  int64_t ldc, c_step;
  void* gu;
  int64_t ldgu;
  int64_t n_out;
  const float* resid;
  void* ws;
  size_t ws_bytes;
};

// ---- few rows an expert -----------------------------------------------------
//
// With a row or a few tokens an expert, reading the weights is all there is to do,
// and a 128 x 128 tile has too few blocks and too long a K for it. Here a block owns
// 16 rows of an expert and 64 (nt) or 128 (nn) columns, and its W waves share K: step s
// is wave s % W's, a wave's loads go straight to registers (each weight is used
// once a block: nothing is gained by LDS), the next step's in flight while one is
// multiplied, and the waves' sums meet in LDS, in order. v_mfma_f32_16x16x32_bf16
// takes the weights as first operand (lane l: column l % 16, k l / 16 * 8 ..+ 7; sums
// of lane l: columns l / 16 * 4 ..+ 3 of row l % 16), so sums lie 4 columns together.
// nn: a lane's 16 bytes hold 8 columns of one k; of 8 k-rows it makes the operands of
// 8 MFMAs, which take columns 8 apart (one v_perm a register).
// Bound by the weights' bytes: 8 tokens of 8 of 64 experts of 2 x 768 x 2048 40 us (6.6
// TB/s, part of it from the last-level cache; on 128 x 128 tiles 47), one token each of
// 8 experts of 3584 x 4864 34 (72). Where a long K has few columns beside it there are
// fewer blocks than CUs, and a block's steps bound it: 8 tokens of 2 of 8 experts of 896 x
// 4864 22 us, 14 at the weights' rate.
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 mfma16(u32x4 w, u32x4 x, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), c, 0, 0, 0);
}

constexpr int few_cols(bool b_kmajor) { return b_kmajor ? 64 : 128; }

template <int W, bool B_KMAJOR, int EPI, bool OUT_BF16, class P>
__global__ __launch_bounds__(64 * W) void few_rows_kernel(P p) {
  constexpr int COLS = few_cols(B_KMAJOR), ROWS = 16, STEP = B_KMAJOR ? 64 : 32;
  constexpr int NX = B_KMAJOR ? 2 : 1;  // 16-byte loads of a row's k a step (of weights: 8)
  constexpr int NC = B_KMAJOR ? 4 : 8;  // accumulators
  __shared__ float red[W][ROWS][COLS + 4];
  int bm, bn;
  if (!enter<ROWS, COLS, true, OUT_BF16>(p, blockIdx.x, bm, bn)) return;  // (the whole block)
  const int m0 = bm * ROWS, n0 = bn * COLS;
  const int lane = threadIdx.x & 63, wave = wave_id(), r = lane & 15, q = lane >> 4;

  int64_t x_row = min(m0 + r, p.M - 1);
  if constexpr (P::kIndexed) x_row = min(max(p.index[x_row], 0), static_cast<int>(p.a_rows - 1));
  const uint16_t* const x = p.A + x_row * p.lda + q * 8;
  const uint16_t* w[B_KMAJOR ? 4 : 1];
  if constexpr (B_KMAJOR) {
#pragma unroll
    for (int c = 0; c < 4; ++c) w[c] = p.B + static_cast<int64_t>(min(n0 + c * 16 + r, p.N - 1)) * p.ldb + q * 8;
  } else {
    w[0] = p.B + static_cast<int64_t>(q * 8) * p.ldb + min(n0 + r * 8, p.N - 8);
  }
  f32x4 acc[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) acc[c] = f32x4{};

  u32x4 wv[2][8], xv[2][NX];
  auto load = [&](int step, int slot) __attribute__((always_inline)) {
    const int64_t k = static_cast<int64_t>(step) * STEP;
    if constexpr (B_KMAJOR) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) wv[slot][2 * c + h] = *reinterpret_cast<const u32x4*>(w[c] + k + 32 * h);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) wv[slot][i] = *reinterpret_cast<const u32x4*>(w[0] + (k + i) * p.ldb);
    }
#pragma unroll
    for (int h = 0; h < NX; ++h) xv[slot][h] = *reinterpret_cast<const u32x4*>(x + k + 32 * h);
  };
  auto multiply = [&](int slot) __attribute__((always_inline)) {
    if constexpr (B_KMAJOR) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] = mfma16(wv[slot][2 * c + h], xv[slot][h], acc[c]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u32x4 op;  // column j of the 8 k-rows
#pragma unroll
        for (int i = 0; i < 4; ++i)
          op[i] = __builtin_amdgcn_perm(wv[slot][2 * i + 1][j >> 1], wv[slot][2 * i][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
        acc[j] = mfma16(op, xv[slot][0], acc[j]);
      }
    }
  };
  const int steps = p.K / STEP;
  if (wave < steps) load(wave, 0);
  for (int s = wave; s < steps; s += 2 * W) {
    if (s + W < steps) load(s + W, 1);
    multiply(0);
    if (s + W < steps) {
      if (s + 2 * W < steps) load(s + 2 * W, 0);
      multiply(1);
    }
  }
  if constexpr (B_KMAJOR) {
#pragma unroll
    for (int c = 0; c < 4; ++c) *reinterpret_cast<f32x4*>(&red[wave][r][c * 16 + q * 4]) = acc[c];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<f32x4*>(&red[wave][r][(q * 4 + e) * 8 + 4 * h]) =
            f32x4{acc[4 * h][e], acc[4 * h + 1][e], acc[4 * h + 2][e], acc[4 * h + 3][e]};
  }
  __syncthreads();
  auto sum = [&](int row, int col) __attribute__((always_inline)) {
    f32x4 v = *reinterpret_cast<const f32x4*>(&red[0][row][col]);
#pragma unroll
    for (int i = 1; i < W; ++i) v += *reinterpret_cast<const f32x4*>(&red[i][row][col]);
    return v;
  };
  auto pack4 = [](f32x4 v) { return make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])); };
  constexpr int OUT = EPI == EPI_SWIGLU ? COLS / 2 : COLS;  // columns that leave
  for (int i = threadIdx.x; i < ROWS * OUT / 4; i += 64 * W) {
    const int row = i / (OUT / 4), col = i % (OUT / 4) * 4;
    if (m0 + row >= p.M) break;
    if constexpr (EPI == EPI_SWIGLU) {
      const int n = n0 / 2 + col;
      if (n >= p.n_out) continue;  // (n_out is a multiple of 32, as the block's columns are)
      const f32x4 g = sum(row, col), u = sum(row, col + 32);
      f32x4 a;
#pragma unroll
      for (int k = 0; k < 4; ++k) a[k] = silu(g[k]) * u[k];
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.C) + (m0 + row) * p.ldc + n) = pack4(a);
      if (p.gu) {
        uint16_t* const o = p.gu + (m0 + row) * p.ldgu + n0 + col;
        *reinterpret_cast<uint2*>(o) = pack4(g);
        *reinterpret_cast<uint2*>(o + 32) = pack4(u);
      }
    } else {
      const int n = n0 + col;
      if (n >= p.N) continue;  // (N is a multiple of 8)
      const f32x4 v = sum(row, col);
      if constexpr (EPI == EPI_SWIGLU_BWD) {
        const int at = (n >> 5) * 64 + (n & 31);
        const uint16_t* const gu = p.gu + (m0 + row) * p.ldgu + at;
        const uint2 gv = *reinterpret_cast<const uint2*>(gu), uv = *reinterpret_cast<const uint2*>(gu + 32);
        f32x4 dg, du;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t gw = k < 2 ? gv.x : gv.y, uw = k < 2 ? uv.x : uv.y;
          const float g = __uint_as_float((k & 1) ? (gw & 0xffff0000u) : (gw << 16));
          const float u = __uint_as_float((k & 1) ? (uw & 0xffff0000u) : (uw << 16));
          const float sg = sigmoid(g);
          dg[k] = v[k] * u * (sg * (1.0f + g * (1.0f - sg)));
          du[k] = v[k] * g * sg;
        }
        uint16_t* const o = static_cast<uint16_t*>(p.C) + (m0 + row) * p.ldc + at;
        *reinterpret_cast<uint2*>(o) = pack4(dg);
        *reinterpret_cast<uint2*>(o + 32) = pack4(du);
      } else if constexpr (OUT_BF16) {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.C) + (m0 + row) * p.ldc + n) = pack4(v);
      } else {
        *reinterpret_cast<f32x4*>(static_cast<float*>(p.C) + (m0 + row) * p.ldc + n) = v;
      }
    }
  }
}

template <bool INDEXED>
GroupedParams<INDEXED> params(const Grouped& g) {
  GroupedParams<INDEXED> p{};
  p.M = static_cast<int>(g.M);
  p.N = static_cast<int>(g.N);
  p.K = static_cast<int>(g.K);
  p.A = static_cast<const uint16_t*>(g.A);
  p.lda = g.lda;
  p.B = static_cast<const uint16_t*>(g.B);
  p.ldb = g.ldb;
  p.n_out = static_cast<int>(g.n_out);
  p.C = g.C;
  p.ldc = g.ldc;
  p.resid = g.resid;
  p.ldr = g.ldc;
  p.gu = static_cast<uint16_t*>(g.gu);
  p.ldgu = g.ldgu;
  p.ksplit = 1;
  p.offsets = g.offsets;
  p.experts = static_cast<int>(g.experts);
  p.index = g.index;
  p.a_rows = g.a_rows;
  p.b_step = g.b_step;
  p.c_step = g.c_step;
  return p;
}

// The tiles of the worst case: every expert but for one with a row in a tile of its own.
int64_t tiles_of(bool ak, int64_t bm, int64_t bn, int64_t experts, int64_t M, int64_t N) {
  const int64_t grid_n = (N + bn - 1) / bn;
  if (!ak) return ((M + bm - 1) / bm * grid_n + 7) / 8 * 8 * experts;  // (eighths: see enter)
  return (M / bm + (experts < M ? experts : M)) * grid_n;
}

// The same without the blocks that even out eighths: the tiles that have partials.
int64_t real_tiles_of(bool ak, int64_t bm, int64_t bn, int64_t experts, int64_t M, int64_t N) {
  return ak ? tiles_of(ak, bm, bn, experts, M, N) : ((M + bm - 1) / bm) * ((N + bn - 1) / bn) * experts;
}

// How a grouped product runs. The row counts are on the device alone, so this goes by
// their average; half a tile's rows of an expert's last tile are taken to be empty. Rows
// that all go to one expert cost less than the same number dealt evenly, whichever way
// is taken: gate/up of 2 x 768 x 2048, 64 experts, 256 rows (FEW) 21 and 71 us, 512 rows
// (FEW) 31 and 73, 4096 (SMALL) 31 and 96, 131072 of 128 experts (BIG) 650 and 685.
// FEW (few_rows_kernel): at most 4 rows an expert, or 14 where 128 x 128 tiles make less
//   than three rounds of them, or no more of its blocks than two a CU (64 experts of 2 x
//   768 x 2048: 4 rows 59 us, on tiles 87; 10 rows 70 and 91; 32 rows 142 and 97).
// SMALL, BIG: 128 x 128 tiles, two a CU, cut along K where that pays for the partials'
//   round trip, or 256 x 256, whichever is expected to take less. Up to a round of
//   either the ungrouped products' times hold; over more, tiles of unlike length overlap
//   and it is their number that counts, with part of a round for the ends. Measured on
//   460 products of 2 .. 128 experts and 40 rows and more an expert, by both: the one
//   chosen is on average 0.8 % slower than the faster one, small tiles alone 5 %, large
//   alone 25 % (8 experts of 4096 rows, 1024 x 9728: 495 us on large tiles; 125 of 439,
//   3136 x 512: 283, on small 368; 35 experts of 493 rows' 448 x 1024 gradients: 62 and 44).
enum Way { FEW, SMALL_TILES, BIG_TILES };
struct GroupedPlan {
  Way way;
  int split;  // SMALL_TILES: blocks along K of a tile
};
GroupedPlan grouped_plan(bool ak, bool bkm, int64_t experts, int64_t M, int64_t N, int64_t K, Output o) {
  const int64_t used = ak && M < experts ? M : experts;
  int64_t KT = K / BK;
  double small, big;
  if (ak) {
    const double rows = static_cast<double>(M) / used;
    const int64_t few = tiles_of(ak, 16, few_cols(bkm), experts, M, N);
    if (M <= 4 * experts || (M <= 14 * experts && tiles_of(ak, 128, 128, experts, M, N) < 1536) ||
        (M <= 128 * experts && few <= 512))
      return {FEW, 1};
    small = used * (rows / 128 + 0.5 > 1 ? rows / 128 + 0.5 : 1.0) * ((N + 127) / 128);
    big = used * (rows / 256 + 0.5 > 1 ? rows / 256 + 0.5 : 1.0) * ((N + 255) / 256);
  } else {
    KT = (K / experts + BK - 1) / BK;
    small = static_cast<double>(real_tiles_of(ak, 128, 128, experts, M, N));
    big = static_cast<double>(real_tiles_of(ak, 256, 256, experts, M, N));
  }
  if (KT < 1) KT = 1;
  auto whole = [](double tiles) { return static_cast<int64_t>(tiles + 0.999); };
  const int kt = static_cast<int>(KT);
  double t_small = small_time(512, kt, o) * (1.28 * small / 512 + 0.27);
  if (small <= 512) t_small = small_time(whole(small), kt, o);
  double t_big = (big_time(256, kt, 1, o) + 0.1 * big_time(256, 0, 1, o)) * (big / 256 + 0.63);
  if (big <= 256) t_big = big_time(whole(big), kt, 1, o);
  if (!ak && small >= 4096) t_big *= 0.8;  // (short sums: the outputs' bytes, which small tiles write less well)
  int split = 1;
  for (int sp = 2; sp <= 64 && sp * 4 <= KT && small * sp <= 512; ++sp) {
    const double t = small_time(whole(small * sp), static_cast<int>((KT + sp - 1) / sp), o) + 3.0 + 0.02 * small * sp;
    if (t < t_small) {
      t_small = t;
      split = sp;
    }
  }
  return t_big < t_small ? GroupedPlan{BIG_TILES, 1} : GroupedPlan{SMALL_TILES, split};
}
int64_t split_bytes_of(bool ak, int64_t experts, int64_t M, int64_t N, int split) {
  return split > 1 ? real_tiles_of(ak, 128, 128, experts, M, N) * split * (128ll * 128 * 4) : 0;
}

template <bool AK, bool BKM, int EPI, bool OB, bool INDEXED>
int launch_grouped(const char* fn, const Grouped& g, hipStream_t s) {
  using G = GroupedParams<INDEXED>;
  G p = params<INDEXED>(g);
  constexpr Output o = EPI == EPI_SWIGLU ? OUT_SWIGLU : EPI == EPI_SWIGLU_BWD ? OUT_SWIGLU_BWD : EPI == EPI_RESID ? OUT_RESID
                       : OB ? OUT_B16 : OUT_F32;
  const GroupedPlan plan = grouped_plan(AK, BKM, g.experts, g.M, g.N, g.K, o);
  const Way way = plan.way;
  int split = plan.split;
  if (!g.ws || static_cast<int64_t>(g.ws_bytes) < split_bytes_of(AK, g.experts, g.M, g.N, split)) split = 1;
  const int bm = way == FEW ? 16 : way == BIG_TILES ? 256 : 128;
  const int bn = way == FEW ? few_cols(BKM) : bm;
  const int64_t tiles = tiles_of(AK, bm, bn, g.experts, g.M, g.N);
  constexpr int PER_TILE = 4 * (is_swiglu(EPI) ? 2 : 4);  // blocks of a tile's reduction
  if (too_many_blocks(tiles, 64 * kWaves) || (split > 1 && (too_many_blocks(tiles * split, kThreads) || too_many_blocks(tiles * PER_TILE, 256))))
    return fail(MR_EINVAL, "%s: too large", fn);
  dim3 grid(static_cast<unsigned>(tiles));
  if (way == FEW) {
    if constexpr (AK) {
      // (eight waves share a K of 1024 and more, of nt alone: their sums of 128 columns would fill half the LDS)
      if (BKM && g.K >= 1024)
        hipLaunchKernelGGL((few_rows_kernel<BKM ? 8 : 4, BKM, EPI, OB, G>), grid, dim3(64 * (BKM ? 8 : 4)), 0, s, p);
      else
        hipLaunchKernelGGL((few_rows_kernel<4, BKM, EPI, OB, G>), grid, dim3(64 * 4), 0, s, p);
    }
  } else if (way == BIG_TILES) {
    hipLaunchKernelGGL((gemm4_kernel<AK, BKM, EPI, OB, G>), grid, dim3(64 * kWaves4), 0, s, p);
  } else {
    p.ksplit = split;
    p.ws = static_cast<float*>(g.ws);
    grid.x *= split;
    hipLaunchKernelGGL((gemm_kernel<128, 128, AK, BKM, EPI, OB, G>), grid, dim3(kThreads), 0, s, p);
    if (split > 1)
      hipLaunchKernelGGL((gemm_reduce<128, 128, EPI, OB, AK, G>), dim3(static_cast<unsigned>(tiles) * PER_TILE), dim3(256), 0, s, p);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MR_OK : hip_fail(e, fn);
}

// What every grouped product asks of its sizes and of the operands that share a
// rule; es is the size of C's elements.
int check_grouped(const char* fn, const Grouped& g, bool ak, bool bkm, int es) {
  if (g.N % 8 || (ak ? g.K % BK || g.K <= 0 : g.M % 8))
    return fail(MR_EINVAL, ak ? "%s: N must be a multiple of 8 and K a positive multiple of 64 (N=%lld K=%lld)"
                              : "%s: N and M must be multiples of 8 (N=%lld M=%lld)",
                fn, static_cast<long long>(g.N), static_cast<long long>(ak ? g.K : g.M));
  // (K in whole k-tiles is a 31-bit number too; tiles of that many rows are more than a launch has)
  if (g.M > 0x7fffffff || g.N > 0x7fffffff || g.K > 0x7fffffff - (BK - 1) || g.experts > 0x7ffffffe)
    return fail(MR_EINVAL, "%s: too large", fn);
  if (g.lda > kMaxLd || g.ldb > kMaxLd || g.ldc > kMaxLd || g.ldgu > kMaxLd)
    return fail(MR_EINVAL, "%s: leading dimensions above %d are not supported", fn, kMaxLd);
  if (g.lda < (ak ? g.K : g.M) || g.ldb < (bkm ? g.K : g.N))
    return fail(MR_EINVAL, "%s: a leading dimension is smaller than its row", fn);
  if (!ok16(g.A, g.lda) || !ok16(g.B, g.ldb) || g.b_step % 8)
    return fail(MR_EINVAL, "%s: operands must be 16-byte aligned with leading dimensions and experts' steps multiples "
                "of 8", fn);
  if (!aligned16(g.C) || g.ldc * es % 16 || g.c_step * es % 16 || (g.gu && !ok16(g.gu, g.ldgu)))
    return fail(MR_EINVAL, "%s: outputs must be 16-byte aligned with 16-byte rows", fn);
  if (reinterpret_cast<uintptr_t>(g.offsets) % 4 || reinterpret_cast<uintptr_t>(g.index) % 4)
    return fail(MR_EINVAL, "%s: a pointer is not aligned to its elements", fn);
  if (!aligned16(g.ws)) return fail(MR_EINVAL, "%s: workspace must be 16-byte aligned", fn);
  if (g.index && (g.a_rows <= 0 || g.a_rows > 0x7fffffff || span_bytes(g.a_rows, g.lda, g.K, 2) > 0xffffffffll))
    return fail(MR_EINVAL, "%s: rows at an index must lie within 4 GiB (%lld rows of %lld)", fn,
                static_cast<long long>(g.a_rows), static_cast<long long>(g.lda));
  return MR_OK;
}

int64_t all_rows_bytes(int64_t experts, int64_t step, int64_t rows, int64_t ld, int64_t width, int64_t es) {
  return (experts - 1) * step * es + span_bytes(rows, ld, width, es);
}

}  // namespace
}  // namespace mr

extern "C" {

size_t mr_gemm_experts_workspace_bytes(int layout, int output, int64_t experts, int64_t M, int64_t N, int64_t K) {
  int way, split;
  size_t bytes = 0;
  return mr_gemm_experts_plan(layout, output, experts, M, N, K, &way, &split, &bytes) == MR_OK ? bytes : 0;
}

int mr_gemm_experts_plan(int layout, int output, int64_t experts, int64_t M, int64_t N, int64_t K, int* way_out,
                         int* split_out, size_t* workspace_out) {
  using namespace mr;
  clear_error();
  if (layout < 0 || layout > 2 || output < MR_OUT_F32 || output > MR_OUT_SWIGLU_BWD || output == MR_OUT_SWIGLU_SPLIT)
    return fail(MR_EINVAL, "mr_gemm_experts_plan: unknown layout %d or output %d", layout, output);
  if (!way_out || !split_out || !workspace_out) return fail(MR_EINVAL, "mr_gemm_experts_plan: null output");
  *way_out = MR_EXPERTS_FEW;
  *split_out = 1;
  *workspace_out = 0;
  if (experts <= 0 || M < 0 || N < 0 || K < 0) return fail(MR_EINVAL, "mr_gemm_experts_plan: no experts, or a negative size");
  if (experts > 0x7ffffffe || M > 0x7fffffff || N > 0x7fffffff || K > 0x7fffffff)
    return fail(MR_EINVAL, "mr_gemm_experts_plan: too large");
  if (M == 0 || N == 0) return MR_OK;
  constexpr Output kinds[] = {OUT_F32, OUT_B16, OUT_RESID, OUT_SWIGLU, OUT_F32, OUT_SWIGLU_BWD};
  const bool ak = layout != MR_TN;
  const GroupedPlan plan = grouped_plan(ak, layout == MR_NT, experts, M, N, K, kinds[output]);
  *way_out = plan.way == FEW ? MR_EXPERTS_FEW : plan.way == SMALL_TILES ? MR_EXPERTS_SMALL : MR_EXPERTS_LARGE;
  *split_out = plan.split;
  *workspace_out = static_cast<size_t>(split_bytes_of(ak, experts, M, N, plan.split));
  return MR_OK;
}

int mr_gemm_experts(int layout, int64_t experts, int64_t M, int64_t N, int64_t K, const void* A, int64_t lda,
                    const int32_t* index, int64_t a_rows, const void* B, int64_t ldb, int64_t b_step,
                    const int32_t* offsets, void* C, int c_dtype, int64_t ldc, int64_t c_step, int accumulate,
                    void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mr;
  clear_error();
  const char* fn = "mr_gemm_experts";
  if (layout < 0 || layout > 2) return fail(MR_EINVAL, "%s: unknown layout %d", fn, layout);
  if (experts <= 0 || M < 0 || N < 0 || K < 0) return fail(MR_EINVAL, "%s: no experts, or a negative size", fn);
  if (c_dtype != MR_F32 && c_dtype != MR_BF16) return fail(MR_EINVAL, "%s: C must be fp32 or bf16", fn);
  const bool tn = layout == MR_TN, ob = c_dtype == MR_BF16;
  if (index && layout != MR_NT) return fail(MR_EINVAL, "%s: only the rows of an nt product may lie at an index", fn);
  if (tn && ob) return fail(MR_EINVAL, "%s: weight gradients are fp32", fn);
  if (accumulate && !tn) return fail(MR_EINVAL, "%s: only weight gradients are added to what is there", fn);
  if (M == 0 || N == 0) return MR_OK;
  if (!offsets || !C || ((!A || !B) && (!tn || K))) return fail(MR_EINVAL, "%s: null operand", fn);
  Grouped g{};
  g.ws = workspace_bytes ? workspace : nullptr;
  g.ws_bytes = workspace_bytes;
  g.M = M;
  g.N = N;
  g.K = K;
  g.A = A;
  g.lda = lda;
  g.index = index;
  g.a_rows = a_rows;
  g.B = B;
  g.ldb = ldb;
  g.b_step = tn ? 0 : b_step;
  g.offsets = offsets;
  g.experts = experts;
  g.C = C;
  g.ldc = ldc;
  g.c_step = tn ? c_step : 0;
  const int es = ob ? 2 : 4;
  if (ldc < N) return fail(MR_EINVAL, "%s: a leading dimension is smaller than its row", fn);
  if (const int rc = check_grouped(fn, g, !tn, layout == MR_NT, es)) return rc;
  const int64_t b_rows = layout == MR_NT ? N : K, b_cols = layout == MR_NT ? K : N;
  if (tn ? c_step < (M - 1) * ldc + N : experts > 1 && b_step < (b_rows - 1) * ldb + b_cols)
    return fail(MR_EINVAL, "%s: the experts' matrices overlap", fn);
  {
    const Region w[2] = {{g.ws, static_cast<int64_t>(g.ws_bytes)}, {C, tn ? all_rows_bytes(experts, c_step, M, ldc, N, 4) : span_bytes(M, ldc, N, es)}};
    const Region r[4] = {{A, tn ? span_bytes(K, lda, M, 2) : span_bytes(index ? a_rows : M, lda, K, 2)},
                         {B, tn ? span_bytes(K, ldb, N, 2) : all_rows_bytes(experts, b_step, b_rows, ldb, b_cols, 2)},
                         {offsets, (experts + 1) * 4},
                         {index, M * 4}};
    if (writes_overlap(w, r)) return fail(MR_EINVAL, "%s: C and the workspace must not overlap what is read or each other", fn);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (layout == MR_NT) {
    if (index)
      return ob ? launch_grouped<true, true, EPI_STORE, true, true>(fn, g, s)
                : launch_grouped<true, true, EPI_STORE, false, true>(fn, g, s);
    return ob ? launch_grouped<true, true, EPI_STORE, true, false>(fn, g, s)
              : launch_grouped<true, true, EPI_STORE, false, false>(fn, g, s);
  }
  if (layout == MR_NN)
    return ob ? launch_grouped<true, false, EPI_STORE, true, false>(fn, g, s)
              : launch_grouped<true, false, EPI_STORE, false, false>(fn, g, s);
  if (!accumulate) return launch_grouped<false, false, EPI_STORE, false, false>(fn, g, s);
  g.resid = static_cast<const float*>(C);
  return launch_grouped<false, false, EPI_RESID, false, false>(fn, g, s);
}

int mr_gemm_experts_swiglu(int64_t experts, int64_t M, int64_t N, int64_t K, const void* X, int64_t ldx,
                           const int32_t* index, int64_t x_rows, const void* Wgu, int64_t ldw, int64_t w_step,
                           const int32_t* offsets, void* act, int64_t ldact, void* gu, int64_t ldgu,
                           void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mr;
  clear_error();
  const char* fn = "mr_gemm_experts_swiglu";
  if (experts <= 0 || M < 0 || N < 0 || K < 0) return fail(MR_EINVAL, "%s: no experts, or a negative size", fn);
  if (M == 0 || N == 0) return MR_OK;
  if (!X || !Wgu || !offsets || !act) return fail(MR_EINVAL, "%s: null operand", fn);
  if (N % 32) return fail(MR_EINVAL, "%s: N must be a multiple of 32 (N=%lld)", fn, static_cast<long long>(N));
  Grouped g{};
  g.ws = workspace_bytes ? workspace : nullptr;
  g.ws_bytes = workspace_bytes;
  g.M = M;
  g.N = 2 * N;
  g.n_out = N;
  g.K = K;
  g.A = X;
  g.lda = ldx;
  g.index = index;
  g.a_rows = x_rows;
  g.B = Wgu;
  g.ldb = ldw;
  g.b_step = w_step;
  g.offsets = offsets;
  g.experts = experts;
  g.C = act;
  g.ldc = ldact;
  g.gu = gu;
  g.ldgu = gu ? ldgu : 0;
  if (ldact < N || (gu && ldgu < 2 * N)) return fail(MR_EINVAL, "%s: a leading dimension is smaller than its row", fn);
  if (const int rc = check_grouped(fn, g, true, true, 2)) return rc;
  if (experts > 1 && w_step < (2 * N - 1) * ldw + K) return fail(MR_EINVAL, "%s: the experts' matrices overlap", fn);
  {
    const Region w[3] = {{g.ws, static_cast<int64_t>(g.ws_bytes)}, {act, span_bytes(M, ldact, N, 2)}, {gu, gu ? span_bytes(M, ldgu, 2 * N, 2) : 0}};
    const Region r[4] = {{X, span_bytes(index ? x_rows : M, ldx, K, 2)},
                         {Wgu, all_rows_bytes(experts, w_step, 2 * N, ldw, K, 2)},
                         {offsets, (experts + 1) * 4},
                         {index, M * 4}};
    if (writes_overlap(w, r)) return fail(MR_EINVAL, "%s: act, gu and the workspace must not overlap what is read or each other", fn);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  return index ? launch_grouped<true, true, EPI_SWIGLU, true, true>(fn, g, s)
               : launch_grouped<true, true, EPI_SWIGLU, true, false>(fn, g, s);
}

int mr_gemm_experts_swiglu_bwd(int64_t experts, int64_t M, int64_t N, int64_t K, const void* dy, int64_t ldd,
                               const void* Wd, int64_t ldw, int64_t w_step, const int32_t* offsets, const void* gu,
                               int64_t ldgu, void* dgu, int64_t lddgu, void* workspace, size_t workspace_bytes,
                               void* stream) {
  using namespace mr;
  clear_error();
  const char* fn = "mr_gemm_experts_swiglu_bwd";
  if (experts <= 0 || M < 0 || N < 0 || K < 0) return fail(MR_EINVAL, "%s: no experts, or a negative size", fn);
  if (M == 0 || N == 0) return MR_OK;
  if (!dy || !Wd || !offsets || !gu || !dgu) return fail(MR_EINVAL, "%s: null operand", fn);
  if (N % 32) return fail(MR_EINVAL, "%s: N must be a multiple of 32 (N=%lld)", fn, static_cast<long long>(N));
  Grouped g{};
  g.ws = workspace_bytes ? workspace : nullptr;
  g.ws_bytes = workspace_bytes;
  g.M = M;
  g.N = N;
  g.K = K;
  g.A = dy;
  g.lda = ldd;
  g.B = Wd;
  g.ldb = ldw;
  g.b_step = w_step;
  g.offsets = offsets;
  g.experts = experts;
  g.C = dgu;
  g.ldc = lddgu;
  g.gu = const_cast<void*>(gu);
  g.ldgu = ldgu;
  if (ldgu < 2 * N || lddgu < 2 * N) return fail(MR_EINVAL, "%s: a leading dimension is smaller than its row", fn);
  if (const int rc = check_grouped(fn, g, true, false, 2)) return rc;
  if (experts > 1 && w_step < (K - 1) * ldw + N) return fail(MR_EINVAL, "%s: the experts' matrices overlap", fn);
  {
    // dgu may be written over gu itself: the lane that writes a piece has read it
    const bool in_place = dgu == gu && lddgu == ldgu;
    const Region w[2] = {{g.ws, static_cast<int64_t>(g.ws_bytes)}, {dgu, span_bytes(M, lddgu, 2 * N, 2)}};
    const Region r[4] = {{dy, span_bytes(M, ldd, K, 2)},
                         {Wd, all_rows_bytes(experts, w_step, K, ldw, N, 2)},
                         {offsets, (experts + 1) * 4},
                         {in_place ? nullptr : gu, span_bytes(M, ldgu, 2 * N, 2)}};
    if (writes_overlap(w, r) || (in_place && g.ws && overlap(g.ws, g.ws_bytes, gu, span_bytes(M, ldgu, 2 * N, 2))))
      return fail(MR_EINVAL, "%s: dgu and the workspace must not overlap what is read (unless dgu is gu itself) or each "
                  "other", fn);
  }
  return launch_grouped<true, false, EPI_SWIGLU_BWD, true, false>(fn, g, static_cast<hipStream_t>(stream));
}

}  // extern "C"
