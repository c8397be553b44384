// The bf16 products' entry points: plain, residual and SwiGLU outputs. The tiles,
// epilogues and plans are mr_gemm_tiles.h's.
#include "mr_gemm_tiles.h"

namespace mr {
namespace {

// mr_gemm_swiglu, or with `split` (rows of 3N) mr_gemm_swiglu_split, where
// act is optional.
int swiglu_product(const char* fn, int64_t M, int64_t N, int64_t K, const void* X, int64_t ldx, const void* Wgu,
                   int64_t ldw, void* split, int64_t ldsplit, void* act, int64_t ldact, void* gu, int64_t ldgu,
                   void* workspace, size_t workspace_bytes, void* stream) {
  if (M <= 0 || N <= 0) return MR_OK;
  if (!X || !Wgu || (!act && !split)) return fail(MR_EINVAL, "%s: null operand", fn);
  if (M % 8 || N % 32 || K % BK || K <= 0)
    return fail(MR_EINVAL, "%s: M %% 8, N %% 32 and K %% %d must be 0", fn, BK);
  if (!ok16(X, ldx) || !ok16(Wgu, ldw) || (act && !ok16(act, ldact)) || (gu && !ok16(gu, ldgu)) ||
      (split && !ok16(split, ldsplit)))
    return fail(MR_EINVAL, "%s: operands and outputs must be 16-byte aligned with leading "
                "dimensions multiples of 8", fn);
  if (ldx < K || ldw < K || (act && ldact < N) || (gu && ldgu < 2 * N) || (split && ldsplit < 3 * N) || ldx > kMaxLd ||
      ldw > kMaxLd || (act && ldact > kMaxLd) || (gu && ldgu > kMaxLd) || (split && ldsplit > kMaxLd))
    return fail(MR_EINVAL, "%s: bad leading dimension", fn);
  {
    const Region w[4] = {{act, act ? span_bytes(M, ldact, N, 2) : 0}, {gu, gu ? span_bytes(M, ldgu, 2 * N, 2) : 0},
                         {split, split ? span_bytes(M, ldsplit, 3 * N, 2) : 0},
                         {workspace, static_cast<int64_t>(workspace_bytes)}};
    const Region r[2] = {{X, span_bytes(M, ldx, K, 2)}, {Wgu, span_bytes(2 * N, ldw, K, 2)}};
    if (writes_overlap(w, r))
      return fail(MR_EINVAL, "%s: act, gu and the workspace must not overlap X, Wgu or each other", fn);
  }
  GemmParams p{};
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(2 * N);
  p.n_out = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.A = static_cast<const uint16_t*>(X);
  p.lda = ldx;
  p.B = static_cast<const uint16_t*>(Wgu);
  p.ldb = ldw;
  p.C = split ? split : act;
  p.ldc = split ? ldsplit : ldact;
  p.gu = static_cast<uint16_t*>(gu);
  p.ldgu = ldgu;
  if (!set_workspace(p, workspace, workspace_bytes))
    return fail(MR_EINVAL, "%s: workspace must be 16-byte aligned", fn);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (!split) return dispatch<true, true, EPI_SWIGLU, true>(p, s);
  p.act = static_cast<uint16_t*>(act);
  p.ldact = ldact;
  return dispatch<true, true, EPI_SWIGLU_SPLIT, true>(p, s);
}

}  // namespace
}  // namespace mr

extern "C" {

size_t mr_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return static_cast<size_t>(mr::split_bytes(M, N, K));
}

int mr_gemm_plan(int layout, int output, int64_t M, int64_t N, int64_t K, size_t workspace_bytes, int* tiles_out,
                 int* split_out, int64_t* tail_out) {
  using namespace mr;
  clear_error();
  if (layout < 0 || layout > 2 || output < MR_OUT_F32 || output > MR_OUT_SWIGLU_BWD)
    return fail(MR_EINVAL, "mr_gemm_plan: unknown layout %d or output %d", layout, output);
  if (M <= 0 || N <= 0 || K <= 0 || K % BK || M > 0x7fffffff || N > 0x7fffffff || K > 0x7fffffff)
    return fail(MR_EINVAL, "mr_gemm_plan: M and N positive, K a positive multiple of %d", BK);
  if (!tiles_out || !split_out || !tail_out) return fail(MR_EINVAL, "mr_gemm_plan: null output");
  constexpr Output kinds[] = {OUT_F32, OUT_B16, OUT_RESID, OUT_SWIGLU, OUT_F32, OUT_SWIGLU_BWD};
  const int KT = static_cast<int>(K / BK);
  const int64_t ws = static_cast<int64_t>(workspace_bytes < kSplitCapBytes ? workspace_bytes : kSplitCapBytes);
  const Plan p = plan_for(M, N, KT, layout != MR_TN, kinds[output], ws);
  const int64_t bm = p.kind == BIG || p.kind == WIDE ? 256 : 128, bn = p.kind == BIG ? 256 : 128;
  const int64_t tiles = ((M + bm - 1) / bm) * ((N + bn - 1) / bn);
  int split = p.kind == BIG ? split_plan(tiles, KT, ws) : p.split;
  if (p.kind != SMALL && split > 1) split = (KT + (KT + split - 1) / split - 1) / ((KT + split - 1) / split);  // no empty split
  const bool quarters = p.kind == BIG && (output <= MR_OUT_BF16 || output == MR_OUT_SWIGLU_SPLIT) && quarter_tail(tiles, split);
  *tiles_out = p.kind == BIG ? (quarters ? MR_TILES_LARGE_QUARTERS : MR_TILES_LARGE)
                             : p.kind == SMALL ? MR_TILES_SMALL : p.kind == DEEP ? MR_TILES_DEEP : MR_TILES_WIDE;
  *split_out = split;
  *tail_out = p.kind == SMALL ? tiles : tiles % 256;
  return MR_OK;
}

int mr_gemm(int layout, int64_t M, int64_t N, int64_t K, const void* A, int64_t lda,
            const void* B, int64_t ldb, void* C, int c_dtype, int64_t ldc, const float* bias,
            const float* resid, int64_t ldr, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mr;
  clear_error();
  if (M < 0 || N < 0 || K < 0) return fail(MR_EINVAL, "mr_gemm: negative size");
  if (M == 0 || N == 0) return MR_OK;
  if (!A || !B || !C) return fail(MR_EINVAL, "mr_gemm: null operand");
  if (M % 8 || N % 8 || K % BK || K == 0)
    return fail(MR_EINVAL, "mr_gemm: M and N must be multiples of 8 and K a positive multiple of %d "
                "(M=%lld N=%lld K=%lld)", BK, (long long)M, (long long)N, (long long)K);
  if (M > 0x7fffffff || N > 0x7fffffff || K > 0x7fffffff) return fail(MR_EINVAL, "mr_gemm: too large");
  if (lda > kMaxLd || ldb > kMaxLd || ldc > kMaxLd || (resid && ldr > kMaxLd))
    return fail(MR_EINVAL, "mr_gemm: leading dimensions above %d are not supported", kMaxLd);
  if (!ok16(A, lda) || !ok16(B, ldb))
    return fail(MR_EINVAL, "mr_gemm: operands must be 16-byte aligned with ld a multiple of 8");
  if (c_dtype != MR_F32 && c_dtype != MR_BF16) return fail(MR_EINVAL, "mr_gemm: C must be fp32 or bf16");
  if (!aligned16(C) || ldc % (c_dtype == MR_BF16 ? 8 : 4) || (resid && (!aligned16(resid) || ldr % 4)))
    return fail(MR_EINVAL, "mr_gemm: C and resid must be 16-byte aligned with 16-byte rows");
  if (resid && c_dtype != MR_F32) return fail(MR_EINVAL, "mr_gemm: the residual form writes fp32");
  if (layout < 0 || layout > 2) return fail(MR_EINVAL, "mr_gemm: unknown layout %d", layout);
  {
    const bool a_kmajor = layout != 2, b_kmajor = layout == 0;
    if (lda < (a_kmajor ? K : M) || ldb < (b_kmajor ? K : N) || ldc < N || (resid && ldr < N))
      return fail(MR_EINVAL, "mr_gemm: a leading dimension is smaller than its row");
    // C may be the residual itself (same place, same rows), nothing else it reads
    const int64_t nc = span_bytes(M, ldc, N, c_dtype == MR_BF16 ? 2 : 4);
    const bool in_place = resid == C && ldr == ldc;
    const Region w[2] = {{C, nc}, {workspace, static_cast<int64_t>(workspace_bytes)}};
    const Region r[3] = {{A, a_kmajor ? span_bytes(M, lda, K, 2) : span_bytes(K, lda, M, 2)},
                         {B, b_kmajor ? span_bytes(N, ldb, K, 2) : span_bytes(K, ldb, N, 2)},
                         {in_place ? nullptr : resid, resid ? span_bytes(M, ldr, N, 4) : 0}};
    if (writes_overlap(w, r) || (in_place && workspace && overlap(workspace, workspace_bytes, C, nc)))
      return fail(MR_EINVAL, "mr_gemm: C and the workspace must not overlap A, B, the residual (unless C is "
                  "the residual itself) or each other");
  }
  GemmParams p{};
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.A = static_cast<const uint16_t*>(A);
  p.lda = lda;
  p.B = static_cast<const uint16_t*>(B);
  p.ldb = ldb;
  p.C = C;
  p.ldc = ldc;
  p.bias = bias;
  p.resid = resid;
  p.ldr = ldr;
  if (!set_workspace(p, workspace, workspace_bytes))
    return fail(MR_EINVAL, "mr_gemm: workspace must be 16-byte aligned");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool ob = c_dtype == MR_BF16;
#define MR_GEMM_CASE(AK, BKM)                                                             \
  if (resid) return dispatch<AK, BKM, EPI_RESID, false>(p, s);                            \
  return ob ? dispatch<AK, BKM, EPI_STORE, true>(p, s)                                    \
            : dispatch<AK, BKM, EPI_STORE, false>(p, s);
  switch (layout) {
    case 0: { MR_GEMM_CASE(true, true) }    // NT: Y = X W^T
    case 1: { MR_GEMM_CASE(true, false) }   // NN: dX = dY W
    case 2: { MR_GEMM_CASE(false, false) }  // TN: dW = dY^T X
    default: return fail(MR_EINVAL, "mr_gemm: unknown layout %d", layout);
  }
#undef MR_GEMM_CASE
}

int mr_gemm_swiglu(int64_t M, int64_t N, int64_t K, const void* X, int64_t ldx, const void* Wgu,
                   int64_t ldw, void* act, int64_t ldact, void* gu, int64_t ldgu, void* workspace,
                   size_t workspace_bytes, void* stream) {
  mr::clear_error();
  return mr::swiglu_product("mr_gemm_swiglu", M, N, K, X, ldx, Wgu, ldw, nullptr, 0, act, ldact, gu, ldgu, workspace,
                            workspace_bytes, stream);
}

int mr_gemm_swiglu_split(int64_t M, int64_t N, int64_t K, const void* X, int64_t ldx, const void* Wgu,
                         int64_t ldw, void* act_split, int64_t ldsplit, void* act, int64_t ldact, void* gu,
                         int64_t ldgu, void* workspace, size_t workspace_bytes, void* stream) {
  mr::clear_error();
  if (M <= 0 || N <= 0) return MR_OK;
  if (!act_split) return mr::fail(MR_EINVAL, "mr_gemm_swiglu_split: null operand");
  if (!act != !gu) return mr::fail(MR_EINVAL, "mr_gemm_swiglu_split: act and gu come together");
  return mr::swiglu_product("mr_gemm_swiglu_split", M, N, K, X, ldx, Wgu, ldw, act_split, ldsplit, act, ldact, gu,
                            ldgu, workspace, workspace_bytes, stream);
}

int mr_gemm_swiglu_bwd(int64_t M, int64_t N, int64_t K, const void* dd, int64_t ldd,
                       const void* Wd, int64_t ldw, const void* gu, int64_t ldgu, void* dgu,
                       int64_t lddgu, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mr;
  clear_error();
  if (M <= 0 || N <= 0) return MR_OK;
  if (!dd || !Wd || !gu || !dgu) return fail(MR_EINVAL, "mr_gemm_swiglu_bwd: null operand");
  if (M % 8 || N % 32 || K % BK || K == 0)
    return fail(MR_EINVAL, "mr_gemm_swiglu_bwd: M %% 8, N %% 32 and K %% %d must be 0", BK);
  if (!ok16(dd, ldd) || !ok16(Wd, ldw) || !ok16(gu, ldgu) || !ok16(dgu, lddgu))
    return fail(MR_EINVAL, "mr_gemm_swiglu_bwd: operands and gu/dgu must be 16-byte aligned with leading "
                "dimensions multiples of 8");
  if (ldd < K || ldw < N || lddgu < 2 * N || ldd > kMaxLd || ldw > kMaxLd || lddgu > kMaxLd)
    return fail(MR_EINVAL, "mr_gemm_swiglu_bwd: bad leading dimension");
  if (ldgu != lddgu) return fail(MR_EINVAL, "mr_gemm_swiglu_bwd: gu and dgu must share a layout");
  {
    // dgu may be written over gu itself: each piece of gu is read before the
    // same piece of dgu is written, by the same lane
    const int64_t ng = span_bytes(M, ldgu, 2 * N, 2);
    const Region w[2] = {{dgu, ng}, {workspace, static_cast<int64_t>(workspace_bytes)}};
    const Region r[3] = {{dd, span_bytes(M, ldd, K, 2)}, {Wd, span_bytes(K, ldw, N, 2)},
                         {dgu == gu ? nullptr : gu, ng}};
    if (writes_overlap(w, r) || (dgu == gu && workspace && overlap(workspace, workspace_bytes, gu, ng)))
      return fail(MR_EINVAL, "mr_gemm_swiglu_bwd: dgu and the workspace must not overlap dd, Wd, gu (unless dgu "
                  "is gu itself) or each other");
  }
  GemmParams p{};
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.A = static_cast<const uint16_t*>(dd);
  p.lda = ldd;
  p.B = static_cast<const uint16_t*>(Wd);
  p.ldb = ldw;
  p.C = dgu;
  p.ldc = lddgu;
  p.gu = const_cast<uint16_t*>(static_cast<const uint16_t*>(gu));
  p.ldgu = ldgu;
  if (!set_workspace(p, workspace, workspace_bytes))
    return fail(MR_EINVAL, "mr_gemm_swiglu_bwd: workspace must be 16-byte aligned");
  return dispatch<true, false, EPI_SWIGLU_BWD, true>(p, static_cast<hipStream_t>(stream));
}

}  // extern "C"
