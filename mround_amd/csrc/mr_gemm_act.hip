// Products with an activation in their epilogue, for ungated MLPs and residual
// branches, and their backward:
//   forward   C = f(X W^T + bias) (+ resid),  pre = X W^T + bias
//   backward  dpre = (dd Wd) f'(pre)  from the next product's output gradient dd,
//             dpre = dout f'(pre)     from the output's own gradient,
//             dbias = column sums of dpre.
// dX = dpre W and dW = dpre^T X are the plain products. The tiles, the plans and
// the epilogues are mr_gemm_tiles.h's: what f costs is the epilogue's time, in the
// product's last microseconds, where an output in fp32 and a pass of its own would
// write and read it again.
//
// Bound by the matrix cores: silu of 16384 x 18944 x 3584 with the pre-activation
// saved takes 1758 to 1843 us (1207 to 1265 TFLOP/s, by the card). At 4096 x 11008 x
// 2048, where the products alone take 146 us forward and 149 backward, they take with
// these epilogues 159 (relu) to 182 us (erf gelu) and 165 to 184 with the
// pre-activation saved; backward 161 to 185, of which reading the pre-activation is 12
// and the erf gelu's slope 24, and a bias gradient 6 to 7 more. A slice of 32 rows
// reads what its epilogue needs when it starts, with nothing beside it to cover the wait.
#include "mr_gemm_tiles.h"

namespace mr {
namespace {

template <int F>
int act_forward(const GemmParams& p, bool bf16, hipStream_t s) {
  return bf16 ? dispatch<true, true, EPI_ACT + F, true>(p, s) : dispatch<true, true, EPI_ACT + F, false>(p, s);
}

// dpre = dout f'(pre) over 32 rows and 256 columns a block (32 lanes of 8 columns, a
// wave 2 rows at a time and 8 in all, all of a thread's loads in flight), and the
// rows' column sums. Bound by memory; blocks of 512 columns left 4 waves a CU at
// 4005 x 896.
template <int F, int DT>
__global__ __launch_bounds__(256) void act_bwd_rows(const void* dout, int64_t ldo, const uint16_t* pre,
                                                    int64_t ldpre, uint16_t* dpre, int64_t ldd, int64_t M, int N,
                                                    float* colsum) {
  __shared__ float part[4][256];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * 32 + wave * 8 + (lane >> 5);
  const int col = blockIdx.x * 256 + (lane & 31) * 8, cb = min(col, N - 8);
  float d[4][8], x[4][8];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int64_t row = row0 + 2 * r < M ? row0 + 2 * r : M - 1;
    load8<DT>(dout, row * ldo + cb, d[r]);
    load8<MR_BF16>(pre, row * ldpre + cb, x[r]);
  }
  float sums[8] = {};
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (row0 + 2 * r >= M || col >= N) continue;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      d[r][k] *= activate_slope<F>(x[r][k]);
      sums[k] += d[r][k];
    }
    store8<MR_BF16>(dpre, (row0 + 2 * r) * ldd + col, d[r]);
  }
  if (!colsum) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    sums[k] += __shfl_xor(sums[k], 32, 64);
    if (lane < 32) part[wave][lane * 8 + k] = sums[k];
  }
  __syncthreads();
  const int c = threadIdx.x;
  if (static_cast<int>(blockIdx.x) * 256 + c < N)
    colsum[static_cast<int64_t>(blockIdx.y) * N + blockIdx.x * 256 + c] = part[0][c] + part[1][c] + part[2][c] + part[3][c];
}

// dbias: the column sums of 32 rows each, added up in a fixed order. A block takes
// 64 columns, 16 waves every sixteenth row of sums.
__global__ __launch_bounds__(1024) void sum_columns(const float* __restrict__ colsum, int rows, int N,
                                                    float* __restrict__ dbias) {
  __shared__ float part[16][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = blockIdx.x * 64 + lane;
  float s = 0.0f;
  if (col < N) {
#pragma unroll 8
    for (int r = wave; r < rows; r += 16) s += colsum[static_cast<int64_t>(r) * N + col];
  }
  part[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && col < N) {
#pragma unroll
    for (int w = 1; w < 16; ++w) s += part[w][lane];
    dbias[col] = s;
  }
}

bool valid_act(int act) { return act >= MR_ACT_RELU && act <= MR_ACT_GELU_TANH; }
int64_t partial_bytes(int64_t M, int64_t N) { return (M + 31) / 32 * N * 4; }

int add_bias_gradient(const char* fn, const float* partials, int64_t M, int64_t N, float* dbias, hipStream_t s) {
  hipLaunchKernelGGL(sum_columns, dim3(static_cast<unsigned>((N + 63) / 64)), dim3(1024), 0, s, partials,
                     static_cast<int>((M + 31) / 32), static_cast<int>(N), dbias);
  MR_LAUNCH_CHECK(fn);
  return MR_OK;
}

// What both backward entry points ask of dbias and its partial sums.
int check_bias_gradient(const char* fn, int64_t M, int64_t N, const float* dbias, const float* partials, size_t bytes) {
  if (!dbias) return MR_OK;
  if (too_many_blocks((N + 63) / 64, 1024)) return fail(MR_EINVAL, "%s: too large, N=%lld", fn, static_cast<long long>(N));
  if (!partials || static_cast<int64_t>(bytes) < partial_bytes(M, N))
    return fail(MR_EINVAL, "%s: dbias needs %lld bytes of partials", fn, static_cast<long long>(partial_bytes(M, N)));
  if (!aligned16(partials) || reinterpret_cast<uintptr_t>(dbias) % 4)
    return fail(MR_EINVAL, "%s: partials must be 16-byte aligned, dbias aligned to its elements", fn);
  return MR_OK;
}

}  // namespace
}  // namespace mr

#define MR_ACT_CASES(CALL)                       \
  switch (act) {                                 \
    case MR_ACT_RELU: CALL(MR_ACT_RELU);         \
    case MR_ACT_RELU2: CALL(MR_ACT_RELU2);       \
    case MR_ACT_SILU: CALL(MR_ACT_SILU);         \
    case MR_ACT_GELU: CALL(MR_ACT_GELU);         \
    default: CALL(MR_ACT_GELU_TANH);             \
  }

extern "C" {

size_t mr_bias_partials_bytes(int64_t M, int64_t N) {
  return M <= 0 || N <= 0 ? 0 : static_cast<size_t>(mr::partial_bytes(M, N));
}

int mr_gemm_act(int64_t M, int64_t N, int64_t K, const void* X, int64_t ldx, const void* W, int64_t ldw, int act,
                const float* bias, const float* resid, int64_t ldr, void* C, int c_dtype, int64_t ldc, void* pre,
                int64_t ldpre, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mr;
  clear_error();
  if (M < 0 || N < 0 || K < 0) return fail(MR_EINVAL, "mr_gemm_act: negative size");
  if (!valid_act(act)) return fail(MR_EINVAL, "mr_gemm_act: unknown activation %d", act);
  if (M == 0 || N == 0) return MR_OK;
  if (!X || !W || !C) return fail(MR_EINVAL, "mr_gemm_act: null operand");
  if (N % 8 || K % BK || K == 0)
    return fail(MR_EINVAL, "mr_gemm_act: N must be a multiple of 8 and K a positive multiple of %d (N=%lld K=%lld)", BK,
                static_cast<long long>(N), static_cast<long long>(K));
  if (M > 0x7fffffff || N > 0x7fffffff || K > 0x7fffffff) return fail(MR_EINVAL, "mr_gemm_act: too large");
  if (c_dtype != MR_F32 && c_dtype != MR_BF16) return fail(MR_EINVAL, "mr_gemm_act: C must be fp32 or bf16");
  if (resid && c_dtype != MR_F32) return fail(MR_EINVAL, "mr_gemm_act: the residual form writes fp32");
  if (ldx < K || ldw < K || ldc < N || (resid && ldr < N) || (pre && ldpre < N))
    return fail(MR_EINVAL, "mr_gemm_act: a leading dimension is smaller than its row");
  if (ldx > kMaxLd || ldw > kMaxLd || ldc > kMaxLd || (resid && ldr > kMaxLd) || (pre && ldpre > kMaxLd))
    return fail(MR_EINVAL, "mr_gemm_act: leading dimensions above %d are not supported", kMaxLd);
  if (!ok16(X, ldx) || !ok16(W, ldw) || (pre && !ok16(pre, ldpre)))
    return fail(MR_EINVAL, "mr_gemm_act: X, W and pre must be 16-byte aligned with leading dimensions multiples of 8");
  if (!aligned16(C) || ldc % (c_dtype == MR_BF16 ? 8 : 4) || (resid && (!aligned16(resid) || ldr % 4)) ||
      reinterpret_cast<uintptr_t>(bias) % 4)
    return fail(MR_EINVAL, "mr_gemm_act: C and resid must be 16-byte aligned with 16-byte rows, bias to its elements");
  {
    const int64_t nc = span_bytes(M, ldc, N, c_dtype == MR_BF16 ? 2 : 4);
    const bool in_place = resid == C && ldr == ldc;
    const Region w[3] = {{C, nc}, {pre, pre ? span_bytes(M, ldpre, N, 2) : 0},
                         {workspace_bytes ? workspace : nullptr, static_cast<int64_t>(workspace_bytes)}};
    const Region r[4] = {{X, span_bytes(M, ldx, K, 2)}, {W, span_bytes(N, ldw, K, 2)}, {bias, N * 4},
                         {in_place ? nullptr : resid, resid ? span_bytes(M, ldr, N, 4) : 0}};
    if (writes_overlap(w, r))
      return fail(MR_EINVAL, "mr_gemm_act: C, pre and the workspace must not overlap X, W, bias, the residual (unless C "
                  "is the residual itself) or each other");
  }
  GemmParams p{};
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.A = static_cast<const uint16_t*>(X);
  p.lda = ldx;
  p.B = static_cast<const uint16_t*>(W);
  p.ldb = ldw;
  p.C = C;
  p.ldc = ldc;
  p.bias = bias;
  p.resid = resid;
  p.ldr = ldr;
  p.pre = static_cast<uint16_t*>(pre);
  p.ldpre = ldpre;
  if (!set_workspace(p, workspace, workspace_bytes))
    return fail(MR_EINVAL, "mr_gemm_act: workspace must be 16-byte aligned");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool bf16 = c_dtype == MR_BF16;
#define MR_FORWARD(F) return act_forward<F>(p, bf16, s)
  MR_ACT_CASES(MR_FORWARD)
#undef MR_FORWARD
}

int mr_gemm_act_bwd(int64_t M, int64_t N, int64_t K, const void* dd, int64_t ldd, const void* Wd, int64_t ldw,
                    const void* pre, int64_t ldpre, int act, void* dpre, int64_t lddpre, float* dbias, float* partials,
                    size_t partials_bytes, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mr;
  clear_error();
  if (M < 0 || N < 0 || K < 0) return fail(MR_EINVAL, "mr_gemm_act_bwd: negative size");
  if (!valid_act(act)) return fail(MR_EINVAL, "mr_gemm_act_bwd: unknown activation %d", act);
  if (N == 0 || (M == 0 && !dbias)) return MR_OK;
  if (M == 0) return fail(MR_EINVAL, "mr_gemm_act_bwd: no rows to sum dbias over");
  if (!dd || !Wd || !pre || !dpre) return fail(MR_EINVAL, "mr_gemm_act_bwd: null operand");
  if (N % 8 || K % BK || K == 0)
    return fail(MR_EINVAL, "mr_gemm_act_bwd: N must be a multiple of 8 and K a positive multiple of %d (N=%lld K=%lld)",
                BK, static_cast<long long>(N), static_cast<long long>(K));
  if (M > 0x7fffffff || N > 0x7fffffff || K > 0x7fffffff) return fail(MR_EINVAL, "mr_gemm_act_bwd: too large");
  if (ldd < K || ldw < N || ldpre < N || lddpre < N)
    return fail(MR_EINVAL, "mr_gemm_act_bwd: a leading dimension is smaller than its row");
  if (ldd > kMaxLd || ldw > kMaxLd || ldpre > kMaxLd || lddpre > kMaxLd)
    return fail(MR_EINVAL, "mr_gemm_act_bwd: leading dimensions above %d are not supported", kMaxLd);
  if (!ok16(dd, ldd) || !ok16(Wd, ldw) || !ok16(pre, ldpre) || !ok16(dpre, lddpre))
    return fail(MR_EINVAL, "mr_gemm_act_bwd: operands and outputs must be 16-byte aligned with leading dimensions "
                "multiples of 8");
  if (const int rc = check_bias_gradient("mr_gemm_act_bwd", M, N, dbias, partials, partials_bytes)) return rc;
  {
    // dpre may be written over pre itself: the lane that writes a piece has read it
    const bool in_place = dpre == pre && lddpre == ldpre;
    const Region w[4] = {{dpre, span_bytes(M, lddpre, N, 2)}, {dbias, N * 4}, {dbias ? partials : nullptr, partial_bytes(M, N)},
                         {workspace_bytes ? workspace : nullptr, static_cast<int64_t>(workspace_bytes)}};
    const Region r[3] = {{dd, span_bytes(M, ldd, K, 2)}, {Wd, span_bytes(K, ldw, N, 2)},
                         {in_place ? nullptr : pre, span_bytes(M, ldpre, N, 2)}};
    if (writes_overlap(w, r))
      return fail(MR_EINVAL, "mr_gemm_act_bwd: dpre, dbias, the partials and the workspace must not overlap dd, Wd, pre "
                  "(unless dpre is pre itself) or each other");
  }
  GemmParams p{};
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.A = static_cast<const uint16_t*>(dd);
  p.lda = ldd;
  p.B = static_cast<const uint16_t*>(Wd);
  p.ldb = ldw;
  p.C = dpre;
  p.ldc = lddpre;
  p.pre = const_cast<uint16_t*>(static_cast<const uint16_t*>(pre));
  p.ldpre = ldpre;
  p.colsum = dbias ? partials : nullptr;
  if (!set_workspace(p, workspace, workspace_bytes))
    return fail(MR_EINVAL, "mr_gemm_act_bwd: workspace must be 16-byte aligned");
  hipStream_t s = static_cast<hipStream_t>(stream);
  int rc = MR_OK;
#define MR_BACKWARD(F) rc = dispatch<true, false, EPI_ACT_BWD + F, true>(p, s); break
  MR_ACT_CASES(MR_BACKWARD)
#undef MR_BACKWARD
  if (rc != MR_OK || !dbias) return rc;
  return add_bias_gradient("mr_gemm_act_bwd", partials, M, N, dbias, s);
}

int mr_act_bwd(int64_t M, int64_t N, const void* dout, int dout_dtype, int64_t ldo, const void* pre, int64_t ldpre, int act,
               void* dpre, int64_t lddpre, float* dbias, float* partials, size_t partials_bytes, void* stream) {
  using namespace mr;
  clear_error();
  if (M < 0 || N < 0) return fail(MR_EINVAL, "mr_act_bwd: negative size");
  if (!valid_act(act)) return fail(MR_EINVAL, "mr_act_bwd: unknown activation %d", act);
  if (dout_dtype != MR_F32 && dout_dtype != MR_BF16) return fail(MR_EINVAL, "mr_act_bwd: dout must be fp32 or bf16");
  if (N == 0 || (M == 0 && !dbias)) return MR_OK;
  if (M == 0) return fail(MR_EINVAL, "mr_act_bwd: no rows to sum dbias over");
  if (!dout || !pre || !dpre) return fail(MR_EINVAL, "mr_act_bwd: null operand");
  if (N % 8) return fail(MR_EINVAL, "mr_act_bwd: N must be a multiple of 8 (N=%lld)", static_cast<long long>(N));
  if (M > 32ll * 65535 || N > 0x7ffffe00) return fail(MR_EINVAL, "mr_act_bwd: too large");
  if (ldo < N || ldpre < N || lddpre < N) return fail(MR_EINVAL, "mr_act_bwd: a leading dimension is smaller than N");
  const int es = dtype_bytes(dout_dtype);
  if (!aligned16(dout) || (ldo * es) % 16 || !ok16(pre, ldpre) || !ok16(dpre, lddpre))
    return fail(MR_EINVAL, "mr_act_bwd: operands and outputs must be 16-byte aligned with 16-byte rows");
  if (const int rc = check_bias_gradient("mr_act_bwd", M, N, dbias, partials, partials_bytes)) return rc;
  {
    // dpre may be written over pre or a bf16 dout itself: the lane that writes a piece has read it
    const bool over_pre = dpre == pre && lddpre == ldpre, over_dout = dpre == dout && lddpre == ldo && es == 2;
    const Region w[3] = {{dpre, span_bytes(M, lddpre, N, 2)}, {dbias, N * 4}, {dbias ? partials : nullptr, partial_bytes(M, N)}};
    const Region r[2] = {{over_dout ? nullptr : dout, span_bytes(M, ldo, N, es)}, {over_pre ? nullptr : pre, span_bytes(M, ldpre, N, 2)}};
    if (writes_overlap(w, r))
      return fail(MR_EINVAL, "mr_act_bwd: dpre, dbias and the partials must not overlap dout, pre (unless dpre is either "
                  "itself) or each other");
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 g(static_cast<unsigned>((N + 255) / 256), static_cast<unsigned>((M + 31) / 32));
  const uint16_t* x = static_cast<const uint16_t*>(pre);
  uint16_t* d = static_cast<uint16_t*>(dpre);
  float* cs = dbias ? partials : nullptr;
#define MR_BACKWARD(F)                                                                                                     \
  if (dout_dtype == MR_F32)                                                                                                \
    hipLaunchKernelGGL((act_bwd_rows<F, MR_F32>), g, dim3(256), 0, s, dout, ldo, x, ldpre, d, lddpre, M, static_cast<int>(N), cs); \
  else                                                                                                                     \
    hipLaunchKernelGGL((act_bwd_rows<F, MR_BF16>), g, dim3(256), 0, s, dout, ldo, x, ldpre, d, lddpre, M, static_cast<int>(N), cs); \
  break
  MR_ACT_CASES(MR_BACKWARD)
#undef MR_BACKWARD
  MR_LAUNCH_CHECK("mr_act_bwd");
  return dbias ? add_bias_gradient("mr_act_bwd", partials, M, N, dbias, s) : MR_OK;
}

}  // extern "C"
