// The norms around a block, fused with its gate and residual scale (gfx950).
//
//   p = post(h)            LayerNorm, RMS norm or nothing, with weight and bias
//   u = p * act(gate)      act: sigmoid, silu or no gate
//   r = x + scale * u      scale a row vector or one number; r = u without x
//   y = pre(r)             the next block's norm, of the sum before it is rounded
//
// Gradients, with n the normalised rows and N'(dn) = rstd (dn - n mean(dn n) [- mean(dn)]):
//   g = dr + N'_pre(dy pre_w);  dx = g;  dscale = sum g u;  du = g scale
//   dgate = du p act'(gate);  dp = du act(gate);  dh = N'_post(dp post_w)
//   dpre_w = sum dy n_pre, dpre_b = sum dy, dpost_w = sum dp n_post, dpost_b = sum dp
//
// Bound by memory: the forward reads h, x, gate and writes r, y; the backward reads h, x,
// gate, dr, dy and writes dh, dx, dgate.  So a row is read once and stays in registers: a
// group of TPR lanes holds it, K vectors of 8 consecutive elements a lane, and the groups
// walk over rows with the row vectors (weights) loaded once.  The backward forms p, u and r
// again from h, x and gate rather than reading them (r, rounded, would cost as many bytes as
// x), from the forward's means and reciprocal deviations (16 bytes a row).
//
// The row vectors' gradients are sums over all rows: every workgroup sums its rows in
// registers, then over its groups in LDS in a fixed order, and writes one partial row; a
// second launch adds the partials in order.  No atomics: results are the same on every run.
//
// Everything between loads and stores is fp32; variances are of the centred values.
#include "mg_common.h"

namespace {

typedef uint16_t u16;

enum { RN_NONE = 0, RN_LAYER = 1, RN_RMS = 2 };
enum { RN_NOGATE = 0, RN_SIGMOID = 1, RN_SILU = 2 };
enum { RN_DSCALE = 0, RN_DPOST_W = 1, RN_DPOST_B = 2, RN_DPRE_W = 3, RN_DPRE_B = 4, RN_NPAR = 5 };

struct RnArgs {
  const void *h, *x, *gate, *scale, *post_w, *post_b, *pre_w, *pre_b;
  int64_t ldh, ldx, ldg, rows;
  float scale_const, eps;
  int D, post, act, pre;
  float4* stats;  // a row's (post mean, post rstd, pre mean, pre rstd), or null
  void *r, *y;
  // backward
  const void *dr, *dy;
  int64_t lddr, lddy;
  void *dh, *dx, *dgate;
  float* part;  // (gridDim.x, RN_NPAR, D) partial sums, or null
};

template <typename E>
struct Vec8;
template <>
struct Vec8<float> {
  float4 a, b;
  __device__ __forceinline__ void get(float (&v)[8]) const {
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    a = make_float4(v[0], v[1], v[2], v[3]);
    b = make_float4(v[4], v[5], v[6], v[7]);
  }
};
template <>
struct Vec8<u16> {
  uint4 q;
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (unsigned)__builtin_bit_cast(u16, (__bf16)v[2 * i]) |
             ((unsigned)__builtin_bit_cast(u16, (__bf16)v[2 * i + 1]) << 16);
    q = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
__device__ __forceinline__ float rn_ld1(const float* p) { return *p; }
__device__ __forceinline__ float rn_ld1(const u16* p) { return __uint_as_float((unsigned)*p << 16); }
__device__ __forceinline__ void rn_st1(float* p, float x) { *p = x; }
__device__ __forceinline__ void rn_st1(u16* p, float x) { *p = __builtin_bit_cast(u16, (__bf16)x); }

// Elements c .. c+7 of a row of D; past D they read as 0 and are not written.  VEC: D and
// every row start are multiples of 16 bytes, so 8 elements lie inside or outside together.
template <typename E, bool VEC>
__device__ __forceinline__ void rn_load(const E* row, int c, int D, float (&v)[8]) {
  if constexpr (VEC) {
    if (c < D) {
      reinterpret_cast<const Vec8<E>*>(row + c)->get(v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < D ? rn_ld1(row + c + i) : 0.f;
  }
}
template <typename E, bool VEC>
__device__ __forceinline__ void rn_store(E* row, int c, int D, const float (&v)[8]) {
  if constexpr (VEC) {
    if (c < D) {
      Vec8<E> q;
      q.set(v);
      *reinterpret_cast<Vec8<E>*>(row + c) = q;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < D) rn_st1(row + c + i, v[i]);
  }
}

// A row's sums over its TPR lanes, in every one of them.  Past one wave the waves' sums meet
// in LDS; `turn` alternates between two sets of slots, so one barrier is enough: a wave can
// be at most one sum ahead of the others.
template <int TPR, int N>
__device__ __forceinline__ void rn_sum(float (&s)[N], int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = mg_group_sum<(TPR < MG_WAVE ? TPR : MG_WAVE)>(s[i]);
  if constexpr (TPR > MG_WAVE) {
    constexpr int W = TPR / MG_WAVE;
    __shared__ float slots[2][4][W];
    const int w = threadIdx.x / MG_WAVE;
    if ((threadIdx.x & (MG_WAVE - 1)) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) slots[turn][i][w] = s[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = 0.f;
#pragma unroll
      for (int j = 0; j < W; ++j) t += slots[turn][i][j];
      s[i] = t;
    }
    turn ^= 1;
  }
}

// Mean and reciprocal deviation of a row held in v (elements past D are 0).
template <int TPR, int K>
__device__ __forceinline__ float2 rn_stats(const float (&v)[K][8], int kind, int c0, int D,
                                           float eps, int& turn) {
  float mean = 0.f;
  if (kind == RN_LAYER) {
    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[0] += v[k][i];
    rn_sum<TPR>(s, turn);
    mean = s[0] / (float)D;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = c0 + k * TPR * 8 + i < D ? v[k][i] - mean : 0.f;
      q[0] += d * d;
    }
  rn_sum<TPR>(q, turn);
  return make_float2(mean, 1.f / sqrtf(q[0] / (float)D + eps));
}

__device__ __forceinline__ float rn_sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

template <int K, typename P, bool VEC, int TPR>
__device__ __forceinline__ void rn_vector(const void* p, float other, int c0, int D,
                                          float (&v)[K][8]) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (p) {
      rn_load<P, VEC>((const P*)p, c0 + k * TPR * 8, D, v[k]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] = other;
    }
  }
}

template <typename E, typename P, int TPR, int K, bool VEC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void residual_norm_fwd(RnArgs a) {
  constexpr int NT = TPR > 256 ? TPR : 256, ROWS = NT / TPR;
  const int c0 = (threadIdx.x % TPR) * 8, D = a.D;
  float scale[K][8], pw[K][8], pb[K][8], qw[K][8], qb[K][8];
  rn_vector<K, P, VEC, TPR>(a.scale, a.scale_const, c0, D, scale);
  rn_vector<K, P, VEC, TPR>(a.post_w, 1.f, c0, D, pw);
  rn_vector<K, P, VEC, TPR>(a.post_b, 0.f, c0, D, pb);
  rn_vector<K, P, VEC, TPR>(a.pre_w, 1.f, c0, D, qw);
  rn_vector<K, P, VEC, TPR>(a.pre_b, 0.f, c0, D, qb);
  int turn = 0;
  // A group past the last row repeats it without storing, so that whole waves stay active.
  for (int64_t base = (int64_t)blockIdx.x * ROWS; base < a.rows; base += (int64_t)gridDim.x * ROWS) {
    const int64_t at = base + threadIdx.x / TPR;
    const bool live = at < a.rows;
    const int64_t row = live ? at : a.rows - 1;
    float u[K][8], xv[K][8], gv[K][8];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = c0 + k * TPR * 8;
      rn_load<E, VEC>((const E*)a.h + row * a.ldh, c, D, u[k]);
      if (a.x) rn_load<E, VEC>((const E*)a.x + row * a.ldx, c, D, xv[k]);
      if (a.act) rn_load<E, VEC>((const E*)a.gate + row * a.ldg, c, D, gv[k]);
    }
    float4 st = make_float4(0.f, 1.f, 0.f, 1.f);
    if (a.post) {
      const float2 m = rn_stats<TPR, K>(u, a.post, c0, D, a.eps, turn);
      st.x = m.x, st.y = m.y;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) u[k][i] = (u[k][i] - m.x) * m.y * pw[k][i] + pb[k][i];
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (a.act) {
          const float s = rn_sigmoid(gv[k][i]);
          u[k][i] *= a.act == RN_SILU ? s * gv[k][i] : s;
        }
        if (a.x) u[k][i] = xv[k][i] + scale[k][i] * u[k][i];
        u[k][i] = c0 + k * TPR * 8 + i < D ? u[k][i] : 0.f;  // not the bias past the row
      }
    if (a.r && live) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        rn_store<E, VEC>((E*)a.r + row * D, c0 + k * TPR * 8, D, u[k]);
    }
    if (a.pre) {
      const float2 m = rn_stats<TPR, K>(u, a.pre, c0, D, a.eps, turn);
      st.z = m.x, st.w = m.y;
      if (live) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
          float y[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = (u[k][i] - m.x) * m.y * qw[k][i] + qb[k][i];
          rn_store<E, VEC>((E*)a.y + row * D, c0 + k * TPR * 8, D, y);
        }
      }
    }
    if (a.stats && live && threadIdx.x % TPR == 0) a.stats[row] = st;
  }
}

template <typename E, typename P, int TPR, int K, bool VEC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void residual_norm_bwd(RnArgs a) {
  constexpr int NT = TPR > 256 ? TPR : 256, ROWS = NT / TPR;
  const int c0 = (threadIdx.x % TPR) * 8, D = a.D;
  const float inv = 1.f / (float)D;
  float scale[K][8], pw[K][8], pb[K][8], qw[K][8];
  rn_vector<K, P, VEC, TPR>(a.scale, a.scale_const, c0, D, scale);
  rn_vector<K, P, VEC, TPR>(a.post_w, 1.f, c0, D, pw);
  rn_vector<K, P, VEC, TPR>(a.post_b, 0.f, c0, D, pb);
  rn_vector<K, P, VEC, TPR>(a.pre_w, 1.f, c0, D, qw);
  // A row of one element: dn (1 - n^2) would cancel down to its rounding; 1 - n^2 = eps rstd^2.
  const auto lone = [&](int kind) { return D == 1 && kind == RN_RMS; };
  float sum[RN_NPAR][K][8];
#pragma unroll
  for (int p = 0; p < RN_NPAR; ++p)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[p][k][i] = 0.f;
  int turn = 0;
  for (int64_t base = (int64_t)blockIdx.x * ROWS; base < a.rows; base += (int64_t)gridDim.x * ROWS) {
    const int64_t at = base + threadIdx.x / TPR;
    const bool live = at < a.rows;
    const int64_t row = live ? at : a.rows - 1;
    float n[K][8], xv[K][8], gv[K][8], g[K][8], dy[K][8];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = c0 + k * TPR * 8;
      rn_load<E, VEC>((const E*)a.h + row * a.ldh, c, D, n[k]);
      if (a.x && a.pre) rn_load<E, VEC>((const E*)a.x + row * a.ldx, c, D, xv[k]);
      if (a.act) rn_load<E, VEC>((const E*)a.gate + row * a.ldg, c, D, gv[k]);
      if (a.dr) {
        rn_load<E, VEC>((const E*)a.dr + row * a.lddr, c, D, g[k]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) g[k][i] = 0.f;
      }
      if (a.dy) rn_load<E, VEC>((const E*)a.dy + row * a.lddy, c, D, dy[k]);
    }
    const float4 st = a.stats ? a.stats[row] : make_float4(0.f, 1.f, 0.f, 1.f);
    if (a.post) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) n[k][i] = (n[k][i] - st.x) * st.y;
    }
    // n, p = n w + b, u = p act(gate), r = x + scale u, formed again where they are used.
    const auto post = [&](int k, int i) { return a.post ? n[k][i] * pw[k][i] + pb[k][i] : n[k][i]; };
    const auto act = [&](int k, int i) {
      if (!a.act) return 1.f;
      const float s = rn_sigmoid(gv[k][i]);
      return a.act == RN_SILU ? s * gv[k][i] : s;
    };
    if (a.dy) {
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u = post(k, i) * act(k, i);
          const float r = a.x ? xv[k][i] + scale[k][i] * u : u;
          xv[k][i] = (r - st.z) * st.w;  // the pre norm's rows
          if (live) {
            sum[RN_DPRE_W][k][i] += dy[k][i] * xv[k][i];
            sum[RN_DPRE_B][k][i] += dy[k][i];
          }
          dy[k][i] *= qw[k][i];
          s[0] += dy[k][i] * xv[k][i];  // dy is 0 past D
          s[1] += dy[k][i];
        }
      rn_sum<TPR>(s, turn);
      const float m0 = s[0] * inv, m1 = a.pre == RN_LAYER ? s[1] * inv : 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float d = dy[k][i] - xv[k][i] * m0 - m1;
          g[k][i] += st.w * (lone(a.pre) ? dy[k][i] * (a.eps * st.w * st.w) : d);
        }
    }
    if (a.dx && live) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        rn_store<E, VEC>((E*)a.dx + row * D, c0 + k * TPR * 8, D, g[k]);
    }
    // g becomes dp; gv becomes the gate's gradient.
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = c0 + k * TPR * 8 + i < D;
        const float p = post(k, i);
        float f = 1.f, slope = 0.f;
        if (a.act) {
          const float sg = rn_sigmoid(gv[k][i]);
          const float ds = sg * (1.f - sg);
          f = a.act == RN_SILU ? sg * gv[k][i] : sg;
          slope = a.act == RN_SILU ? sg + gv[k][i] * ds : ds;
        }
        if (live) sum[RN_DSCALE][k][i] += g[k][i] * (p * f);
        const float du = in ? (a.x ? g[k][i] * scale[k][i] : g[k][i]) : 0.f;
        gv[k][i] = du * p * slope;
        const float dp = du * f;
        if (live) {
          sum[RN_DPOST_W][k][i] += dp * n[k][i];
          sum[RN_DPOST_B][k][i] += dp;
        }
        g[k][i] = a.post ? dp * pw[k][i] : dp;
        s[0] += g[k][i] * n[k][i];
        s[1] += g[k][i];
      }
    if (a.dgate && live) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        rn_store<E, VEC>((E*)a.dgate + row * D, c0 + k * TPR * 8, D, gv[k]);
    }
    if (a.post) {
      rn_sum<TPR>(s, turn);
      const float m0 = s[0] * inv, m1 = a.post == RN_LAYER ? s[1] * inv : 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float d = g[k][i] - n[k][i] * m0 - m1;
          g[k][i] = st.y * (lone(a.post) ? g[k][i] * (a.eps * st.y * st.y) : d);
        }
    }
    if (a.dh && live) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        rn_store<E, VEC>((E*)a.dh + row * D, c0 + k * TPR * 8, D, g[k]);
    }
  }
  if (!a.part) return;
  // Over the workgroup's groups, then one partial row for each workgroup.
  __shared__ float s[ROWS][TPR * 8];
  float* part = a.part + (int64_t)blockIdx.x * RN_NPAR * D;
#pragma unroll
  for (int p = 0; p < RN_NPAR; ++p) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if constexpr (ROWS == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c0 + k * TPR * 8 + i < D) part[p * D + c0 + k * TPR * 8 + i] = sum[p][k][i];
      } else {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) s[threadIdx.x / TPR][c0 + i] = sum[p][k][i];
        __syncthreads();
        for (int c = threadIdx.x; c < TPR * 8; c += NT) {
          float t = 0.f;
#pragma unroll
          for (int j = 0; j < ROWS; ++j) t += s[j][c];
          if (c + k * TPR * 8 < D) part[p * D + c + k * TPR * 8] = t;
        }
      }
    }
  }
}

struct RnOut {
  void* p[RN_NPAR];
};

// out[c] = sum over the partial rows, in order: 4 waves take every fourth row of 64 columns.
template <typename P>
__global__ __launch_bounds__(256) void residual_norm_sums(const float* __restrict__ part,
                                                          RnOut out, int parts, int D) {
  __shared__ float s[4][MG_WAVE];
  const int lane = threadIdx.x & (MG_WAVE - 1), w = threadIdx.x / MG_WAVE;
  P* dst = (P*)out.p[blockIdx.y];
  if (!dst) return;
  const int col = blockIdx.x * MG_WAVE + lane, c = col < D ? col : D - 1;
  const float* src = part + (int64_t)blockIdx.y * D + c;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  int r = w;
  for (; r + 12 < parts; r += 16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] += src[(int64_t)(r + 4 * i) * RN_NPAR * D];
  }
  for (; r < parts; r += 4) a[0] += src[(int64_t)r * RN_NPAR * D];
  s[w][lane] = (a[0] + a[1]) + (a[2] + a[3]);
  __syncthreads();
  if (w == 0 && col < D) rn_st1(dst + col, (s[0][lane] + s[1][lane]) + (s[2][lane] + s[3][lane]));
}

// A row's lanes: the fewest that hold it with two vectors each, so that narrow rows share a
// wave and a wide one has the registers of a workgroup.
int rn_tpr(int64_t D) { return D <= 256 ? 16 : D <= 1024 ? 64 : D <= 4096 ? 256 : 512; }

// Workgroups: enough to fill the chip several times over; each has partial sums to write, so
// the backward takes no more than RN_PARTS.
constexpr int64_t RN_GRID = 4096, RN_PARTS = 1024;
int64_t rn_grid(int64_t rows, int64_t D, int64_t most) {
  const int tpr = rn_tpr(D), per = tpr > 256 ? 1 : 256 / tpr;
  const int64_t n = (rows + per - 1) / per;
  return n < most ? n : most;
}

bool rn_ok(int64_t rows, int64_t D) { return rows >= 1 && D >= 1 && D <= 8192 && rows <= (1ll << 40) / D; }

bool rn_vec(const void* p, int64_t ld, int esize) {
  return !p || (((uintptr_t)p & 15) == 0 && (ld * esize) % 16 == 0);
}

template <typename E, typename P, int TPR, int K, bool VEC>
void rn_launch(const RnArgs& a, bool bwd, unsigned grid, hipStream_t stream) {
  const dim3 nt(TPR > 256 ? TPR : 256);
  if (bwd)
    hipLaunchKernelGGL((residual_norm_bwd<E, P, TPR, K, VEC>), dim3(grid), nt, 0, stream, a);
  else
    hipLaunchKernelGGL((residual_norm_fwd<E, P, TPR, K, VEC>), dim3(grid), nt, 0, stream, a);
}
template <typename E, typename P, int TPR>
void rn_pick(const RnArgs& a, bool vec, bool bwd, unsigned grid, hipStream_t stream) {
  const bool one = a.D <= TPR * 8;
  if (vec && one) rn_launch<E, P, TPR, 1, true>(a, bwd, grid, stream);
  if (vec && !one) rn_launch<E, P, TPR, 2, true>(a, bwd, grid, stream);
  if (!vec && one) rn_launch<E, P, TPR, 1, false>(a, bwd, grid, stream);
  if (!vec && !one) rn_launch<E, P, TPR, 2, false>(a, bwd, grid, stream);
}
template <typename E, typename P>
int rn_run(const RnArgs& a, bool bwd, unsigned grid, hipStream_t stream) {
  const int e = sizeof(E), p = sizeof(P);
  const bool vec = a.D % 8 == 0 && rn_vec(a.h, a.ldh, e) && rn_vec(a.x, a.ldx, e) &&
                   rn_vec(a.gate, a.ldg, e) && rn_vec(a.scale, a.D, p) &&
                   rn_vec(a.post_w, a.D, p) && rn_vec(a.post_b, a.D, p) &&
                   rn_vec(a.pre_w, a.D, p) && rn_vec(a.pre_b, a.D, p) && rn_vec(a.r, a.D, e) &&
                   rn_vec(a.y, a.D, e) && rn_vec(a.dr, a.lddr, e) && rn_vec(a.dy, a.lddy, e) &&
                   rn_vec(a.dh, a.D, e) && rn_vec(a.dx, a.D, e) && rn_vec(a.dgate, a.D, e);
  switch (rn_tpr(a.D)) {
    case 16: rn_pick<E, P, 16>(a, vec, bwd, grid, stream); break;
    case 64: rn_pick<E, P, 64>(a, vec, bwd, grid, stream); break;
    case 256: rn_pick<E, P, 256>(a, vec, bwd, grid, stream); break;
    default: rn_pick<E, P, 512>(a, vec, bwd, grid, stream);
  }
  return hipGetLastError() == hipSuccess ? MG_OK : MG_ERR_LAUNCH;
}
int rn_types(const RnArgs& a, int dtype, int pdtype, bool bwd, unsigned grid, hipStream_t stream) {
  if (dtype == 0) return rn_run<float, float>(a, bwd, grid, stream);
  if (pdtype == 0) return rn_run<u16, float>(a, bwd, grid, stream);
  return rn_run<u16, u16>(a, bwd, grid, stream);
}

bool rn_kinds(int dtype, int pdtype, int post, int act, int pre) {
  return !(dtype & ~1) && !(pdtype & ~1) && (dtype || !pdtype) && post >= 0 && post <= 2 &&
         act >= 0 && act <= 2 && pre >= 0 && pre <= 2;
}

}  // namespace

extern "C" {

size_t mg_residual_norm_workspace_bytes(int64_t rows, int64_t D) {
  return rn_ok(rows, D) ? (size_t)rn_grid(rows, D, RN_PARTS) * RN_NPAR * D * sizeof(float) : 0;
}

int mg_residual_norm_fwd(int dtype, int pdtype, int post, int act, int pre, const void* h,
                         int64_t ldh, const void* x, int64_t ldx, const void* gate, int64_t ldg,
                         const void* scale, float scale_const, const void* post_w,
                         const void* post_b, const void* pre_w, const void* pre_b, void* r,
                         void* y, float* stats, int64_t rows, int64_t D, float eps,
                         hipStream_t stream) {
  if (!h || !rn_kinds(dtype, pdtype, post, act, pre) || !rn_ok(rows, D) || (act && !gate) ||
      (pre && !y) || (!pre && !r) || ldh < D || (x && ldx < D) || (act && ldg < D))
    return MG_ERR_ARG;
  RnArgs a = {};
  a.h = h, a.x = x, a.gate = act ? gate : nullptr, a.scale = scale;
  a.post_w = post_w, a.post_b = post_b, a.pre_w = pre_w, a.pre_b = pre_b;
  a.ldh = ldh, a.ldx = ldx, a.ldg = ldg, a.rows = rows;
  a.scale_const = scale_const, a.eps = eps;
  a.D = (int)D, a.post = post, a.act = act, a.pre = pre;
  a.stats = (float4*)stats, a.r = r, a.y = y;
  return rn_types(a, dtype, pdtype, false, (unsigned)rn_grid(rows, D, RN_GRID), stream);
}

int mg_residual_norm_bwd(int dtype, int pdtype, int post, int act, int pre, const void* h,
                         int64_t ldh, const void* x, int64_t ldx, const void* gate, int64_t ldg,
                         const void* scale, float scale_const, const void* post_w,
                         const void* post_b, const void* pre_w, const float* stats,
                         const void* dr, int64_t lddr, const void* dy, int64_t lddy, void* dh,
                         void* dx, void* dgate, void* dscale, void* dpost_w, void* dpost_b,
                         void* dpre_w, void* dpre_b, int64_t rows, int64_t D, float eps, void* ws,
                         size_t ws_bytes, hipStream_t stream) {
  const bool sums = dscale || dpost_w || dpost_b || dpre_w || dpre_b;
  if (!h || !rn_kinds(dtype, pdtype, post, act, pre) || !rn_ok(rows, D) || (act && !gate) ||
      (dy && !pre) || ((post || pre) && !stats) || ldh < D || (x && ldx < D) ||
      (act && ldg < D) || (dr && lddr < D) || (dy && lddy < D) || (sums && !ws))
    return MG_ERR_ARG;
  if (sums && ws_bytes < mg_residual_norm_workspace_bytes(rows, D)) return MG_ERR_WORKSPACE;
  RnArgs a = {};
  a.h = h, a.x = x, a.gate = act ? gate : nullptr, a.scale = scale;
  a.post_w = post_w, a.post_b = post_b, a.pre_w = pre_w;
  a.ldh = ldh, a.ldx = ldx, a.ldg = ldg, a.rows = rows;
  a.scale_const = scale_const, a.eps = eps;
  a.D = (int)D, a.post = post, a.act = act, a.pre = pre;
  a.stats = (float4*)stats;
  a.dr = dr, a.dy = dy, a.lddr = lddr, a.lddy = lddy;
  a.dh = dh, a.dx = dx, a.dgate = act ? dgate : nullptr;
  a.part = sums ? (float*)ws : nullptr;
  const int64_t grid = rn_grid(rows, D, RN_PARTS);
  const int rc = rn_types(a, dtype, pdtype, true, (unsigned)grid, stream);
  if (rc != MG_OK || !sums) return rc;
  const RnOut out = {{dscale, dpost_w, dpost_b, dpre_w, dpre_b}};
  const dim3 g((unsigned)((D + MG_WAVE - 1) / MG_WAVE), RN_NPAR);
  if (pdtype)
    hipLaunchKernelGGL(residual_norm_sums<u16>, g, dim3(256), 0, stream, a.part, out, (int)grid,
                       (int)D);
  else
    hipLaunchKernelGGL(residual_norm_sums<float>, g, dim3(256), 0, stream, a.part, out, (int)grid,
                       (int)D);
  return hipGetLastError() == hipSuccess ? MG_OK : MG_ERR_LAUNCH;
}

}  // extern "C"
