// The end of a block's branch and the norm that follows it, in one pass:
//
//   n = y rsqrt(mean(y^2) + eps) w_post      (or y itself)
//   h = resid + scale gate n                 (gate of the row's group, or 1)
//   x = h rsqrt(mean(h^2) + eps) w_pre       (optional)
//
// and its backward. With dx the gradient of x, d that of h from elsewhere, and
// rms'(g; v) = r (g - v r^2 mean(g v)) the backward of v r for r = rsqrt(mean(v^2)
// + eps):
//
//   dh = d + rms'(dx w_pre; h)     dresid = dh      dw_pre = sum dx h r_h
//   e = scale dh                   dgate = sum e n  (over the group's rows)
//   b = e gate                     dw_post = sum b y r_y
//   dy = rms'(b w_post; y)
//
// Memory bounds both: a row is read once and held in registers by a block, which
// goes on to other rows with the weights in its registers and the next row's loads
// in flight while it sums the present one (two sums, one after the other). Sums
// over rows stay in the block's registers and leave once a block; a second kernel
// adds the blocks' in order.
#include <cmath>

#include "mr_rows.h"

namespace mr {
namespace {

struct NormParams {
  const void* y;
  int64_t ldy;
  const void* stream;  // resid; in the backward the stream behind the branch, h
  int64_t lds;
  const float* post;
  const float* gate;   // [groups, H], or null
  int64_t gate_rows;   // rows of a group
  const float* pre;
  float scale, eps;
  int64_t T;
  int H;
  void* out;           // h; in the backward dresid
  int64_t ldo;
  void* normed;        // x; in the backward dy
  int64_t ldn;
  // backward
  const void* dx;
  int64_t lddx;
  const void* dout;
  int64_t lddo;
  int64_t chunk, per_group;  // rows of a block; blocks of a group (0: blocks of whole groups)
  int row_threads, teams;    // threads of a row; rows at a time (more than one: a wave each)
  float* part_pre;           // [blocks, H] or null
  float* part_post;
  float* part_gate;          // [groups per_group, H]; per_group 0: dgate itself
};

// A sum over the block, in every thread; `slot` alternates between calls so that one barrier each is enough.
__device__ __forceinline__ float block_sum(float x, float (*smem)[16], int& slot) {
  const float s = wave_sum(x);
  const int waves = blockDim.x >> 6;
  if (waves == 1) return s;
  if ((threadIdx.x & 63) == 0) smem[slot][threadIdx.x >> 6] = s;
  __syncthreads();
  float t = 0.0f;
  for (int i = 0; i < waves; ++i) t += smem[slot][i];
  slot = slot == 2 ? 0 : slot + 1;
  return t;
}

// V columns of a float vector from column c.
template <int V>
__device__ __forceinline__ void load_weights(const float* w, int c, float (&out)[V]) {
  if constexpr (V == 8) {
    load8_f32_cached(w, c, out);
  } else {
    out[0] = w[c];
  }
}

// Thread t holds the pieces t, t + threads, .. (P of them) of its row. As many
// blocks as the card holds go over the rows in turn. Bound by HBM:
// 4005 x 2048 bf16 onto fp32 22.6 us (4.3 TB/s), 16384 x 3584 143 (4.9), 4096 x 16384
// 164 (4.9). Of rows of no whole 16 bytes past 8192 columns the registers of 16 columns a
// thread bound it, 57 to 75 of them spilled: 4096 x 16383 358, x 8191 80.
template <int A, int S, int V, int P, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_fwd(NormParams p) {
  __shared__ float smem[3][16];
  int slot = 0;
  const int threads = blockDim.x;
  const float inv_h = 1.0f / static_cast<float>(p.H);
  int col[P];
  bool in[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    col[i] = (static_cast<int>(threadIdx.x) + i * threads) * V;
    in[i] = col[i] < p.H;
    col[i] = in[i] ? col[i] : 0;
  }
  float wpost[P][V], wpre[P][V], gate[P][V];
#pragma unroll
  for (int i = 0; i < P; ++i) {
#pragma unroll
    for (int k = 0; k < V; ++k) wpost[i][k] = wpre[i][k] = gate[i][k] = 1.0f;
    if (p.post) load_weights<V>(p.post, col[i], wpost[i]);
    if (p.pre) load_weights<V>(p.pre, col[i], wpre[i]);
  }
  Piece<A, V> y[P], y_next[P];
  Piece<S, V> r[P], r_next[P];
  auto fetch = [&](int64_t row) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      y_next[i].load(p.y, row * p.ldy + col[i]);
      r_next[i].load(p.stream, row * p.lds + col[i]);
    }
  };
  int64_t group = -1;
  int64_t row = blockIdx.x;
  if (row < p.T) fetch(row);
  for (; row < p.T; row += gridDim.x) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      y[i] = y_next[i];
      r[i] = r_next[i];
    }
    if (row + gridDim.x < p.T) fetch(row + gridDim.x);
    if (p.gate && row / p.gate_rows != group) {
      group = row / p.gate_rows;
#pragma unroll
      for (int i = 0; i < P; ++i) load_weights<V>(p.gate + group * p.H, col[i], gate[i]);
    }
    float ry = 1.0f;
    if (p.post) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < P; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) ss += in[i] ? y[i].get(k) * y[i].get(k) : 0.0f;
      ry = rsqrtf(block_sum(ss, smem, slot) * inv_h + p.eps);
    }
    float h[P][V];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        h[i][k] = r[i].get(k) + p.scale * (gate[i][k] * (y[i].get(k) * ry * wpost[i][k]));
        ss += in[i] ? h[i][k] * h[i][k] : 0.0f;
      }
      if (in[i]) store_piece<S, V, false>(p.out, row * p.ldo + col[i], h[i]);
    }
    if (p.pre) {
      // (of h before it is rounded to the stream's type)
      const float rh = rsqrtf(block_sum(ss, smem, slot) * inv_h + p.eps);
#pragma unroll
      for (int i = 0; i < P; ++i) {
#pragma unroll
        for (int k = 0; k < V; ++k) h[i][k] = h[i][k] * rh * wpre[i][k];
        if (in[i]) store_piece<A, V, false>(p.normed, row * p.ldn + col[i], h[i]);
      }
    }
  }
}

// Two sums at once, over the `waves` waves of a row.
__device__ __forceinline__ void block_sum2(float& a, float& b, float (*smem)[16][2], int& slot, int waves) {
  a = wave_sum(a);
  b = wave_sum(b);
  if (waves == 1) return;
  if ((threadIdx.x & 63) == 0) {
    smem[slot][threadIdx.x >> 6][0] = a;
    smem[slot][threadIdx.x >> 6][1] = b;
  }
  __syncthreads();
  a = b = 0.0f;
  for (int i = 0; i < waves; ++i) {
    a += smem[slot][i][0];
    b += smem[slot][i][1];
  }
  slot = slot == 2 ? 0 : slot + 1;
}

// Bound by HBM: 16384 x 3584, bf16 and fp32, all gradients 228 us (4.6 TB/s; with an
// accumulator for each gradient, which spilled, 343), 4005 x 2048 41 (28 and the sums'
// launch), 32768 x 256 39 (a row a block 81).
// WHOLE: the block's rows are whole groups of the gate. What dgate and dw_post sum
// differs by factors that are a group's own, dh n: one sum serves both, and the
// factors come in when the group ends.
// The registers of P = 1 are held to those of four waves a SIMD where they fit, two
// rows of up to 512 pieces a CU, with the next row's loads in flight (AHEAD; of 16-bit
// rows onto fp32 5 registers are spilled for it, in the 228 us). Rows past 1024 pieces
// leave no room for that, and registers bound them: a thread of 1024 has 128, and of
// its weights, sums and inputs of 16 columns 116 to 262 are spilled (4096 x 8192 150 us,
// x 8200 408, x 12288 484, x 16384 609, 2.0 TB/s). One column at a time 23 to 114 are
// where a thread holds 8 and 272 to 470 where it holds 16 (4096 x 8191 266 us, x 12287
// 1399, x 16383 1702).
constexpr int waves_for(int A, int V, int P, bool WHOLE) {
  return V == 1 ? 4 : P == 1 ? (A == MR_F32 || WHOLE ? 3 : 4) : 2;
}
template <int A, int S, int V, int P, int THREADS, bool WHOLE>
__global__ __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(waves_for(A, V, P, WHOLE)))) void norm_bwd(NormParams p) {
  constexpr bool AHEAD = THREADS == 512;
  __shared__ float smem[3][16][2];
  int slot = 0;
  const int waves = p.row_threads >> 6, teams = p.teams;
  const int team = teams > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const int thread = static_cast<int>(threadIdx.x) - team * 64;  // in its row
  const float inv_h = 1.0f / static_cast<float>(p.H);
  uint32_t col[P];
  bool in[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = (thread + i * p.row_threads) * V;
    in[i] = c < p.H;
    col[i] = in[i] ? c : 0;
  }
  // this block's rows: a chunk of one group, whose teams take turns, or whole groups,
  // which the teams take in turn
  int64_t row0, row1, group;
  if constexpr (!WHOLE) {
    group = blockIdx.x / p.per_group;
    row0 = group * p.gate_rows + (blockIdx.x % p.per_group) * p.chunk;
    row1 = min(min(row0 + p.chunk, (group + 1) * p.gate_rows), p.T);
  } else {
    row0 = static_cast<int64_t>(blockIdx.x) * p.chunk;
    row1 = min(row0 + p.chunk, p.T);
    group = row0 / p.gate_rows + team;
  }
  row0 += WHOLE ? team * p.gate_rows : team;
  const bool branch = p.post || p.gate;
  float wpre[P][V], c[P][V];  // c = scale gate w_post
  float s_pre[P][V], s[P][V], s_post[P][V];
  auto load_branch = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float w[V];
#pragma unroll
      for (int k = 0; k < V; ++k) c[i][k] = p.scale;
      if (p.gate) {
        load_weights<V>(p.gate + group * p.H, col[i], w);
#pragma unroll
        for (int k = 0; k < V; ++k) c[i][k] *= w[k];
      }
      if (p.post) {
        load_weights<V>(p.post, col[i], w);
#pragma unroll
        for (int k = 0; k < V; ++k) c[i][k] *= w[k];
      }
    }
  };
#pragma unroll
  for (int i = 0; i < P; ++i) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      wpre[i][k] = 1.0f;
      s_pre[i][k] = s[i][k] = s_post[i][k] = 0.0f;
    }
    if (p.pre) load_weights<V>(p.pre, col[i], wpre[i]);
  }
  if (row0 < row1) load_branch();
  // The end of a group: dgate = scale w_post s, and to w_post's gradient scale gate s.
  auto end_group = [&](float* gate_to, int64_t at) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float w[V], o[V];
      if (gate_to) {
#pragma unroll
        for (int k = 0; k < V; ++k) w[k] = 1.0f;
        if (p.post) load_weights<V>(p.post, col[i], w);
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = p.scale * w[k] * s[i][k];
        if (in[i]) store_piece<MR_F32, V, false>(gate_to, at * p.H + col[i], o);
      }
      if (p.part_post) {
#pragma unroll
        for (int k = 0; k < V; ++k) w[k] = 1.0f;
        if (p.gate) load_weights<V>(p.gate + group * p.H, col[i], w);
#pragma unroll
        for (int k = 0; k < V; ++k) s_post[i][k] += p.scale * w[k] * s[i][k];
      }
    }
  };
  Piece<A, V> y[P], y_next[P], g[P], g_next[P];
  Piece<S, V> h[P], h_next[P], d[P], d_next[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    g_next[i].zero();
    h_next[i].zero();
    d_next[i].zero();
    y_next[i].zero();
  }
  constexpr int ea = A == MR_F32 ? 4 : 2, es = S == MR_F32 ? 4 : 2;
  auto fetch = [&](int64_t row) __attribute__((always_inline)) {  // (a row's address is the block's, a lane's offset 32 bits)
    const char* gr = static_cast<const char*>(p.dx) + row * p.lddx * ea;
    const char* hr = static_cast<const char*>(p.stream) + row * p.lds * es;
    const char* dr = static_cast<const char*>(p.dout) + row * p.lddo * es;
    const char* yr = static_cast<const char*>(p.y) + row * p.ldy * ea;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if (p.pre) {
        g_next[i].load(gr, col[i]);
        h_next[i].load(hr, col[i]);
      }
      if (p.dout) d_next[i].load(dr, col[i]);
      if (branch) y_next[i].load(yr, col[i]);
    }
  };
  if (AHEAD && row0 < row1) fetch(row0);
  int64_t left = p.gate_rows;  // WHOLE: rows until the group ends
  for (int64_t row = row0, next; row < row1; row = next) {
    const bool last = WHOLE && (left == 1 || row + 1 == row1);  // of its group
    next = !WHOLE ? row + teams : last ? (group + teams) * p.gate_rows : row + 1;
    if (!AHEAD) fetch(row);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      y[i] = y_next[i];
      g[i] = g_next[i];
      h[i] = h_next[i];
      d[i] = d_next[i];
    }
    if (AHEAD && next < row1) fetch(next);
    float rh = 0.0f, ch = 0.0f;
    if (p.pre) {
      float ss = 0.0f, dot = 0.0f;
#pragma unroll
      for (int i = 0; i < P; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float v = in[i] ? h[i].get(k) : 0.0f;
          ss += v * v;
          dot += g[i].get(k) * wpre[i][k] * v;
        }
      block_sum2(ss, dot, smem, slot, waves);
#pragma unroll
      for (int i = 0; i < P; ++i) g[i].hide();
      rh = rsqrtf(ss * inv_h + p.eps);
      ch = rh * rh * (dot * inv_h);
    }
    float dh[P][V];
    char* const out_row = static_cast<char*>(p.out) + row * p.ldo * es;
#pragma unroll
    for (int i = 0; i < P; ++i) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float v = h[i].get(k), gv = g[i].get(k);
        dh[i][k] = d[i].get(k) + rh * (gv * wpre[i][k] - v * ch);
        s_pre[i][k] += gv * (v * rh);
      }
      if (in[i]) store_piece<S, V, false>(out_row, col[i], dh[i]);
    }
    float ry = 1.0f, cy = 0.0f;
    if (p.post) {
      float ss = 0.0f, dot = 0.0f;
#pragma unroll
      for (int i = 0; i < P; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float v = in[i] ? y[i].get(k) : 0.0f;
          ss += v * v;
          dot += dh[i][k] * c[i][k] * v;
        }
      block_sum2(ss, dot, smem, slot, waves);
#pragma unroll
      for (int i = 0; i < P; ++i) y[i].hide();
      ry = rsqrtf(ss * inv_h + p.eps);
      cy = ry * ry * (dot * inv_h);
    }
    char* const dy_row = static_cast<char*>(p.normed) + row * p.ldn * ea;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float o[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float v = y[i].get(k);  // (without post ry is 1 and cy 0)
        s[i][k] += dh[i][k] * (v * ry);
        o[k] = ry * (dh[i][k] * c[i][k] - v * cy);
      }
      if (in[i]) store_piece<A, V, false>(dy_row, col[i], o);
    }
    if constexpr (WHOLE) {
      --left;
      if (last) {
        end_group(p.part_gate, group);
        if (next < row1) {
          group += teams;
          left = p.gate_rows;
          load_branch();
#pragma unroll
          for (int i = 0; i < P; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) s[i][k] = 0.0f;
        }
      }
    }
  }
  if constexpr (V == 8 && P == 1) {
    if (teams > 1) {  // the first team gets the sums, in order
      __shared__ float each[8][64][8];
      auto meet = [&](float (&x)[P][V]) __attribute__((always_inline)) {
        store_piece<MR_F32, V, false>(&each[team][thread][0], 0, x[0]);
        __syncthreads();
        if (team == 0) {
          for (int t = 1; t < teams; ++t)
#pragma unroll
            for (int k = 0; k < V; ++k) x[0][k] += each[t][thread][k];
        }
        __syncthreads();
      };
      meet(s_pre);
      meet(WHOLE ? s_post : s);
      if (team) return;
    }
  }
  if constexpr (!WHOLE) {
    if (branch) end_group(p.part_gate, blockIdx.x);
  }
#pragma unroll
  for (int i = 0; i < P; ++i) {
    if (!in[i]) continue;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * p.H + col[i];
    if (p.part_pre) store_piece<MR_F32, V, false>(p.part_pre, at, s_pre[i]);
    if (p.part_post) store_piece<MR_F32, V, false>(p.part_post, at, s_post[i]);
  }
}

// out[s, c] = sum over the n rows of part from row s n on, in an order that the
// launch fixes: 64 columns a block, 16 runs of rows (10 sums of 3584 columns over 512
// rows 6 us).
struct SumParams {
  const float* part[3];
  float* out[3];
  int64_t n[3];
  int64_t sums[3];
  int H;
};
__global__ __launch_bounds__(1024) void norm_sum(SumParams p) {
  __shared__ float smem[16][64];
  int which = 0;
  int64_t s = blockIdx.y;
  while (s >= p.sums[which]) s -= p.sums[which++];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
  const int64_t n = p.n[which], per = (n + 15) / 16;
  const int64_t a = w * per, b = min(a + per, n);
  float t = 0.0f;
  if (c < p.H) {
    const float* q = p.part[which] + (s * n + a) * p.H + c;
#pragma unroll 8
    for (int64_t i = a; i < b; ++i, q += p.H) t += *q;
  }
  smem[w][threadIdx.x & 63] = t;
  __syncthreads();
  if (w == 0 && c < p.H) {
#pragma unroll
    for (int i = 1; i < 16; ++i) t += smem[i][threadIdx.x];
    p.out[which][s * p.H + c] = t;
  }
}

constexpr int kMaxH = 16384;
constexpr int64_t kMaxT = int64_t{1} << 40;  // (more than any memory holds; products of sizes stay in 64 bits)
struct Split {
  int64_t chunk, per_group, blocks;
};
// The rows of a backward block: about 512 blocks (two a CU; four, of rows of up to
// 128 threads), each of one group's rows or of whole groups.
Split split_rows(int64_t T, int64_t H, int64_t gate_rows) {
  const int64_t most = H > 512 && H <= 1024 ? 1024 : 512;
  const int64_t want = (T + most - 1) / most;
  if (gate_rows <= want) {
    const int64_t chunk = want / gate_rows * gate_rows;
    return {chunk, 0, (T + chunk - 1) / chunk};
  }
  const int64_t groups = (T + gate_rows - 1) / gate_rows;
  const int64_t per = (gate_rows + want - 1) / want;
  return {(gate_rows + per - 1) / per, per, groups * per};
}

// What a backward's blocks leave for the sums' launch (a gate's rows that one block sums are sums already).
size_t partials_bytes(const Split& sp, int64_t H, bool post, bool gate, bool pre) {
  return static_cast<size_t>((post ? 1 : 0) + (pre ? 1 : 0) + (gate && sp.per_group > 1 ? 1 : 0)) * sp.blocks * H * 4;
}

int check_norm(const char* fn, int64_t T, int64_t H, int act, int stream_type, const float* gate, int64_t gate_rows) {
  if (T < 0 || H < 0) return fail(MR_EINVAL, "%s: negative size", fn);
  if (T > kMaxT) return fail(MR_EINVAL, "%s: too many rows", fn);
  if (!valid_dtype(act) || (stream_type != MR_F32 && stream_type != act))
    return fail(MR_EINVAL, "%s: the stream is fp32 or of the branch's type (%d, %d)", fn, stream_type, act);
  if (H > kMaxH) return fail(MR_EINVAL, "%s: rows of more than %d columns are not supported (%lld)", fn, kMaxH,
                             static_cast<long long>(H));
  if (gate && gate_rows <= 0) return fail(MR_EINVAL, "%s: a gate needs the rows it applies to", fn);
  return MR_OK;
}

bool vector_rows(const void* p, int64_t ld, int es) { return !p || (aligned16(p) && ld * es % 16 == 0); }

// Pieces of a row of n that a thread holds (the kernels' P).
int pieces_a_thread(int n, bool vec) { return vec ? (n > 512 ? 2 : 1) : (n > 8192 ? 16 : n > 4096 ? 8 : 4); }

// threads that hold a row of n pieces, P each
int row_threads(int n, int P) {
  const int t = (n + P - 1) / P;
  return (t + 63) / 64 * 64;
}

int64_t bytes_of(int64_t T, int64_t ld, int64_t H, int es) { return ((T - 1) * ld + H) * es; }

}  // namespace
}  // namespace mr

#define MR_NORM_TYPES(CALL)                                            \
  if (act_dtype == MR_F32) CALL(MR_F32, MR_F32);                       \
  else if (act_dtype == MR_BF16 && stream_dtype == MR_F32) CALL(MR_BF16, MR_F32); \
  else if (act_dtype == MR_BF16) CALL(MR_BF16, MR_BF16);               \
  else if (stream_dtype == MR_F32) CALL(MR_F16, MR_F32);               \
  else CALL(MR_F16, MR_F16)

extern "C" {

int mr_norm_residual(const void* y, int act_dtype, int64_t ldy, const void* resid, int stream_dtype, int64_t ldr,
                     int64_t T, int64_t H, float eps, const float* post, const float* gate, int64_t gate_rows, float scale,
                     const float* pre, void* out, int64_t ldo, void* normed, int64_t ldn, void* stream) {
  using namespace mr;
  clear_error();
  const char* fn = "mr_norm_residual";
  if (const int rc = check_norm(fn, T, H, act_dtype, stream_dtype, gate, gate_rows)) return rc;
  if (T == 0 || H == 0) return MR_OK;
  if (!pre != !normed) return fail(MR_EINVAL, "%s: the next norm's weight and its output come together", fn);
  if (!y || !resid || !out) return fail(MR_EINVAL, "%s: null pointer", fn);
  if (ldy < H || ldr < H || ldo < H || (normed && ldn < H))
    return fail(MR_EINVAL, "%s: a leading dimension is smaller than its row", fn);
  const int ea = dtype_bytes(act_dtype), es = dtype_bytes(stream_dtype);
  if (reinterpret_cast<uintptr_t>(y) % ea || reinterpret_cast<uintptr_t>(normed) % ea ||
      reinterpret_cast<uintptr_t>(resid) % es || reinterpret_cast<uintptr_t>(out) % es ||
      (reinterpret_cast<uintptr_t>(post) | reinterpret_cast<uintptr_t>(gate) | reinterpret_cast<uintptr_t>(pre)) % 4)
    return fail(MR_EINVAL, "%s: a pointer is not aligned to its elements", fn);
  {
    const int64_t no = bytes_of(T, ldo, H, es), nn = normed ? bytes_of(T, ldn, H, ea) : 0;
    const int64_t ny = bytes_of(T, ldy, H, ea), nr = bytes_of(T, ldr, H, es);
    const int64_t ng = gate ? ((T - 1) / gate_rows + 1) * H * 4 : 0;
    auto hit = [&](const void* a, int64_t na, const void* b, int64_t nb) { return a && b && overlap(a, na, b, nb); };
    const bool over_resid = out == resid && ldo == ldr, over_y = normed == y && ldn == ldy;
    bool bad = hit(out, no, y, ny) || (!over_resid && hit(out, no, resid, nr)) || hit(out, no, normed, nn) ||
               (!over_y && hit(normed, nn, y, ny)) || hit(normed, nn, resid, nr);
    for (const void* w : {static_cast<const void*>(post), static_cast<const void*>(pre)})
      bad = bad || hit(out, no, w, H * 4) || hit(normed, nn, w, H * 4);
    bad = bad || hit(out, no, gate, ng) || hit(normed, nn, gate, ng);
    if (bad)
      return fail(MR_EINVAL, "%s: out may be resid and normed may be y; otherwise outputs share no memory with what is "
                  "read or each other", fn);
  }
  NormParams p{};
  p.y = y;
  p.ldy = ldy;
  p.stream = resid;
  p.lds = ldr;
  p.post = post;
  p.gate = gate;
  p.gate_rows = gate ? gate_rows : T;
  p.pre = pre;
  p.scale = scale;
  p.eps = eps;
  p.T = T;
  p.H = static_cast<int>(H);
  p.out = out;
  p.ldo = ldo;
  p.normed = normed;
  p.ldn = ldn;
  const bool vec = H % 8 == 0 && vector_rows(y, ldy, ea) && vector_rows(resid, ldr, es) && vector_rows(out, ldo, es) &&
                   vector_rows(normed, ldn, ea) && vector_rows(post, 0, 4) && vector_rows(pre, 0, 4) && vector_rows(gate, H, 4);
  const int n = static_cast<int>(vec ? H / 8 : H);
  const int P = pieces_a_thread(n, vec);
  const int threads = row_threads(n, P);
  const int64_t most = 256ll * (2048 / threads);
  const dim3 grid(static_cast<unsigned>(T < most ? T : most)), block(threads);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define MR_NORM_LAUNCH(A, S, V, P, N) hipLaunchKernelGGL((norm_fwd<A, S, V, P, N>), grid, block, 0, s, p)
#define MR_NORM(A, S)                                                                             \
  do {                                                                                             \
    if (!vec) {                                                                                   \
      if (n <= 4096) MR_NORM_LAUNCH(A, S, 1, 4, 1024);                                            \
      else if (n <= 8192) MR_NORM_LAUNCH(A, S, 1, 8, 1024);                                       \
      else MR_NORM_LAUNCH(A, S, 1, 16, 1024);                                                     \
    } else if (n <= 512) MR_NORM_LAUNCH(A, S, 8, 1, 512);                                         \
    else if (n <= 1024) MR_NORM_LAUNCH(A, S, 8, 2, 512);                                          \
    else MR_NORM_LAUNCH(A, S, 8, 2, 1024);                                                        \
  } while (0)
  MR_NORM_TYPES(MR_NORM);
#undef MR_NORM
#undef MR_NORM_LAUNCH
  MR_LAUNCH_CHECK(fn);
  return MR_OK;
}

size_t mr_norm_residual_bwd_workspace_bytes(int64_t T, int64_t H, int64_t gate_rows, int post, int gate, int pre) {
  if (T <= 0 || T > mr::kMaxT || H <= 0 || H > mr::kMaxH) return 0;
  const mr::Split sp = mr::split_rows(T, H, gate_rows < 1 ? (gate ? 1 : T) : gate_rows < T ? gate_rows : T);
  size_t n = mr::partials_bytes(sp, H, post, gate, pre);
  // A gate whose gradient is not wanted splits the rows as any other, and none does not.
  if (!gate) {
    const size_t without = mr::partials_bytes(mr::split_rows(T, H, T), H, post, false, pre);
    n = n > without ? n : without;
  }
  return n;
}

int mr_norm_residual_bwd(const void* dnormed, int act_dtype, int64_t lddn, const void* dout, int stream_dtype,
                         int64_t lddo, const void* y, int64_t ldy, const void* out, int64_t ldo, int64_t T, int64_t H,
                         float eps, const float* post, const float* gate, int64_t gate_rows, float scale,
                         const float* pre, void* dy, int64_t lddy, void* dresid, int64_t lddr, float* dpost,
                         float* dgate, float* dpre, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mr;
  clear_error();
  const char* fn = "mr_norm_residual_bwd";
  if (const int rc = check_norm(fn, T, H, act_dtype, stream_dtype, gate, gate_rows)) return rc;
  if (T > 0 && !pre != !dnormed) return fail(MR_EINVAL, "%s: the next norm's weight and its output's gradient come together", fn);
  if ((dpost && !post) || (dgate && !gate) || (dpre && !pre))
    return fail(MR_EINVAL, "%s: a gradient is asked for of a weight that is not there", fn);
  if (T > 0 && !dnormed && !dout) return fail(MR_EINVAL, "%s: no gradient comes in", fn);
  if (H == 0) return MR_OK;
  if (T > 0 && (!dy || !dresid || ((post || gate) && !y) || (pre && !out))) return fail(MR_EINVAL, "%s: null pointer", fn);
  if (T > 0 && (lddy < H || lddr < H || (dnormed && (lddn < H || ldo < H)) || (dout && lddo < H) || ((post || gate) && ldy < H)))
    return fail(MR_EINVAL, "%s: a leading dimension is smaller than its row", fn);
  const int ea = dtype_bytes(act_dtype), es = dtype_bytes(stream_dtype);
  if ((reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(dnormed) | reinterpret_cast<uintptr_t>(dy)) % ea ||
      (reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(dresid)) % es ||
      (reinterpret_cast<uintptr_t>(post) | reinterpret_cast<uintptr_t>(gate) | reinterpret_cast<uintptr_t>(pre) |
       reinterpret_cast<uintptr_t>(dpost) | reinterpret_cast<uintptr_t>(dgate) | reinterpret_cast<uintptr_t>(dpre)) % 4)
    return fail(MR_EINVAL, "%s: a pointer is not aligned to its elements", fn);
  const int64_t rows = T > 0 ? T : 1;
  const int64_t of_gate = gate && gate_rows < rows ? gate_rows : rows;
  const int64_t groups = T > 0 ? (T + of_gate - 1) / of_gate : 0;
  const Split sp = split_rows(rows, H, of_gate);
  const int64_t each = sp.blocks * H * 4;
  const size_t need = T > 0 ? partials_bytes(sp, H, dpost != nullptr, dgate != nullptr, dpre != nullptr) : 0;
  if (need && (!workspace || !aligned16(workspace) || workspace_bytes < need))
    return fail(MR_EINVAL, "%s: %zu bytes of workspace are needed, on an address of 16 bytes", fn, need);
  {
    struct Span { const void* p; int64_t n; };
    const Span wr[6] = {{dy, bytes_of(rows, lddy, H, ea)}, {dresid, bytes_of(rows, lddr, H, es)}, {dpost, H * 4},
                        {dgate, groups * H * 4}, {dpre, H * 4}, {need ? workspace : nullptr, static_cast<int64_t>(need)}};
    const Span rd[7] = {{y, bytes_of(rows, ldy, H, ea)}, {dout, bytes_of(rows, lddo, H, es)}, {dnormed, bytes_of(rows, lddn, H, ea)},
                        {out, bytes_of(rows, ldo, H, es)}, {post, H * 4}, {gate, groups * H * 4}, {pre, H * 4}};
    bool bad = false;
    for (int a = 0; a < 6; ++a) {
      if (!wr[a].p || wr[a].n <= 0) continue;
      for (int b = 0; b < 7; ++b) {
        if (!rd[b].p || rd[b].n <= 0) continue;
        if (a == 0 && b == 0 && dy == y && lddy == ldy) continue;
        if (a == 1 && b == 1 && dresid == dout && lddr == lddo) continue;
        bad = bad || overlap(wr[a].p, wr[a].n, rd[b].p, rd[b].n);
      }
      for (int b = a + 1; b < 6; ++b)
        bad = bad || (wr[b].p && wr[b].n > 0 && overlap(wr[a].p, wr[a].n, wr[b].p, wr[b].n));
    }
    if (bad)
      return fail(MR_EINVAL, "%s: dresid may be dout and dy may be y; otherwise outputs share no memory with what is read "
                  "or each other", fn);
  }
  NormParams p{};
  p.y = y;
  p.ldy = ldy;
  p.stream = out;
  p.lds = ldo;
  p.post = post;
  p.gate = gate;
  p.gate_rows = of_gate;
  p.pre = pre;
  p.scale = scale;
  p.eps = eps;
  p.T = T;
  p.H = static_cast<int>(H);
  p.out = dresid;
  p.ldo = lddr;
  p.normed = dy;
  p.ldn = lddy;
  p.dx = dnormed;
  p.lddx = lddn;
  p.dout = dout;
  p.lddo = lddo;
  p.chunk = sp.chunk;
  p.per_group = sp.per_group;
  char* ws = static_cast<char*>(workspace);
  SumParams q{};
  q.H = p.H;
  int sums = 0;
  int64_t blocks_y = 0;
  auto sum = [&](const float* part, float* to, int64_t n, int64_t count) {
    q.part[sums] = part;
    q.out[sums] = to;
    q.n[sums] = n;
    q.sums[sums++] = count;
    blocks_y += count;
  };
  const int64_t blocks = T > 0 ? sp.blocks : 0;
  if (dpre) {
    p.part_pre = reinterpret_cast<float*>(ws);
    ws += blocks ? each : 0;
    sum(p.part_pre, dpre, blocks, 1);
  }
  if (dpost) {
    p.part_post = reinterpret_cast<float*>(ws);
    ws += blocks ? each : 0;
    sum(p.part_post, dpost, blocks, 1);
  }
  if (dgate && sp.per_group > 1) {
    p.part_gate = reinterpret_cast<float*>(ws);
    if (groups) sum(p.part_gate, dgate, sp.per_group, groups);
  } else {
    p.part_gate = dgate;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (blocks) {
    const bool vec = H % 8 == 0 && vector_rows(y, ldy, ea) && vector_rows(out, ldo, es) && vector_rows(dnormed, lddn, ea) &&
                     vector_rows(dout, lddo, es) && vector_rows(dy, lddy, ea) && vector_rows(dresid, lddr, es) &&
                     vector_rows(post, 0, 4) && vector_rows(pre, 0, 4) && vector_rows(gate, H, 4) && vector_rows(dgate, H, 4);
    const int n = static_cast<int>(vec ? H / 8 : H);
    const int P = pieces_a_thread(n, vec);
    const int threads = row_threads(n, P);
    if (too_many_blocks(blocks, 1024)) return fail(MR_EINVAL, "%s: too many rows", fn);
    // Eight rows at a time where a wave holds one (with one, two waves a CU were all
    // there were: 32768 rows of 256 columns 81 us, 39 now).
    p.row_threads = threads;
    p.teams = vec && threads == 64 ? 8 : 1;
    const dim3 grid(static_cast<unsigned>(blocks)), block(threads * p.teams);
#define MR_NORM_LAUNCH(A, S, V, P, N)                                                              \
  do {                                                                                            \
    if (sp.per_group) hipLaunchKernelGGL((norm_bwd<A, S, V, P, N, false>), grid, block, 0, s, p); \
    else hipLaunchKernelGGL((norm_bwd<A, S, V, P, N, true>), grid, block, 0, s, p);               \
  } while (0)
#define MR_NORM(A, S)                                                                             \
  do {                                                                                             \
    if (!vec) {                                                                                   \
      if (n <= 4096) MR_NORM_LAUNCH(A, S, 1, 4, 1024);                                            \
      else if (n <= 8192) MR_NORM_LAUNCH(A, S, 1, 8, 1024);                                       \
      else MR_NORM_LAUNCH(A, S, 1, 16, 1024);                                                     \
    } else if (n <= 512) MR_NORM_LAUNCH(A, S, 8, 1, 512);                                         \
    else if (n <= 1024) MR_NORM_LAUNCH(A, S, 8, 2, 512);                                          \
    else MR_NORM_LAUNCH(A, S, 8, 2, 1024);                                                        \
  } while (0)
    MR_NORM_TYPES(MR_NORM);
#undef MR_NORM
#undef MR_NORM_LAUNCH
    MR_LAUNCH_CHECK(fn);
  }
  if (blocks_y) {
    // (a gate that several blocks share has more rows than 1/1024 of them: at most 1025 groups)
    hipLaunchKernelGGL(norm_sum, dim3(static_cast<unsigned>((H + 63) / 64), static_cast<unsigned>(blocks_y)), dim3(1024), 0, s, q);
    MR_LAUNCH_CHECK(fn);
  }
  return MR_OK;
}

}  // extern "C"
