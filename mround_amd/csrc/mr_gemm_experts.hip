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
};

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

// The blocks of the worst case: every expert but for one with a row in a tile of its own.
template <int BM, int BN, bool AK>
int64_t blocks_of(const Grouped& g) {
  const int64_t grid_n = (g.N + BN - 1) / BN;
  if (!AK) return (g.M + BM - 1) / BM * grid_n * g.experts;
  return (g.M / BM + (g.experts < g.M ? g.experts : g.M)) * grid_n;
}

template <bool AK, bool BKM, int EPI, bool OB, bool INDEXED>
int launch_grouped(const char* fn, const Grouped& g, hipStream_t s) {
  const GroupedParams<INDEXED> p = params<INDEXED>(g);
  // 256 x 256 tiles where an expert has the rows for one on average, else 128 x 128.
  const bool big = (AK ? g.M / g.experts : g.M) > 128 && g.N > 128;
  const int64_t blocks = big ? blocks_of<256, 256, AK>(g) : blocks_of<128, 128, AK>(g);
  if (too_many_blocks(blocks, kThreads)) return fail(MR_EINVAL, "%s: too large", fn);
  const dim3 grid(static_cast<unsigned>(blocks));
  if (big)
    hipLaunchKernelGGL((gemm4_kernel<AK, BKM, EPI, OB, GroupedParams<INDEXED>>), grid, dim3(64 * kWaves4), 0, s, p);
  else
    hipLaunchKernelGGL((gemm_kernel<128, 128, AK, BKM, EPI, OB, GroupedParams<INDEXED>>), grid, dim3(kThreads), 0, s, p);
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
  if (g.M > 0x7fffffff || g.N > 0x7fffffff || g.K > 0x7fffffff || g.experts > 0x7ffffffe)
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

int mr_gemm_experts(int layout, int64_t experts, int64_t M, int64_t N, int64_t K, const void* A, int64_t lda,
                    const int32_t* index, int64_t a_rows, const void* B, int64_t ldb, int64_t b_step,
                    const int32_t* offsets, void* C, int c_dtype, int64_t ldc, int64_t c_step, int accumulate,
                    void* stream) {
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
    const Region w[1] = {{C, tn ? all_rows_bytes(experts, c_step, M, ldc, N, 4) : span_bytes(M, ldc, N, es)}};
    const Region r[4] = {{A, tn ? span_bytes(K, lda, M, 2) : span_bytes(index ? a_rows : M, lda, K, 2)},
                         {B, tn ? span_bytes(K, ldb, N, 2) : all_rows_bytes(experts, b_step, b_rows, ldb, b_cols, 2)},
                         {offsets, (experts + 1) * 4},
                         {index, M * 4}};
    if (writes_overlap(w, r)) return fail(MR_EINVAL, "%s: C must not overlap what is read", fn);
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
                           const int32_t* offsets, void* act, int64_t ldact, void* gu, int64_t ldgu, void* stream) {
  using namespace mr;
  clear_error();
  const char* fn = "mr_gemm_experts_swiglu";
  if (experts <= 0 || M < 0 || N < 0 || K < 0) return fail(MR_EINVAL, "%s: no experts, or a negative size", fn);
  if (M == 0 || N == 0) return MR_OK;
  if (!X || !Wgu || !offsets || !act) return fail(MR_EINVAL, "%s: null operand", fn);
  if (N % 32) return fail(MR_EINVAL, "%s: N must be a multiple of 32 (N=%lld)", fn, static_cast<long long>(N));
  Grouped g{};
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
    const Region w[2] = {{act, span_bytes(M, ldact, N, 2)}, {gu, gu ? span_bytes(M, ldgu, 2 * N, 2) : 0}};
    const Region r[4] = {{X, span_bytes(index ? x_rows : M, ldx, K, 2)},
                         {Wgu, all_rows_bytes(experts, w_step, 2 * N, ldw, K, 2)},
                         {offsets, (experts + 1) * 4},
                         {index, M * 4}};
    if (writes_overlap(w, r)) return fail(MR_EINVAL, "%s: act and gu must not overlap what is read or each other", fn);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  return index ? launch_grouped<true, true, EPI_SWIGLU, true, true>(fn, g, s)
               : launch_grouped<true, true, EPI_SWIGLU, true, false>(fn, g, s);
}

int mr_gemm_experts_swiglu_bwd(int64_t experts, int64_t M, int64_t N, int64_t K, const void* dy, int64_t ldd,
                               const void* Wd, int64_t ldw, int64_t w_step, const int32_t* offsets, const void* gu,
                               int64_t ldgu, void* dgu, int64_t lddgu, void* stream) {
  using namespace mr;
  clear_error();
  const char* fn = "mr_gemm_experts_swiglu_bwd";
  if (experts <= 0 || M < 0 || N < 0 || K < 0) return fail(MR_EINVAL, "%s: no experts, or a negative size", fn);
  if (M == 0 || N == 0) return MR_OK;
  if (!dy || !Wd || !offsets || !gu || !dgu) return fail(MR_EINVAL, "%s: null operand", fn);
  if (N % 32) return fail(MR_EINVAL, "%s: N must be a multiple of 32 (N=%lld)", fn, static_cast<long long>(N));
  Grouped g{};
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
    const Region w[1] = {{dgu, span_bytes(M, lddgu, 2 * N, 2)}};
    const Region r[4] = {{dy, span_bytes(M, ldd, K, 2)},
                         {Wd, all_rows_bytes(experts, w_step, K, ldw, N, 2)},
                         {offsets, (experts + 1) * 4},
                         {in_place ? nullptr : gu, span_bytes(M, ldgu, 2 * N, 2)}};
    if (writes_overlap(w, r))
      return fail(MR_EINVAL, "%s: dgu must not overlap what is read (unless dgu is gu itself)", fn);
  }
  return launch_grouped<true, false, EPI_SWIGLU_BWD, true, false>(fn, g, static_cast<hipStream_t>(stream));
}

}  // extern "C"
