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
// group of TPR lanes holds it, 8 consecutive elements a lane, and the groups walk over rows.
// The backward forms p, u and r again from h, x and gate rather than reading them (r, rounded,
// would cost as many bytes as x), from the forward's means and reciprocal deviations (16 bytes
// a row).
//
// The row vectors' gradients are sums over all rows: every workgroup sums its rows in
// registers, then over its groups in LDS in a fixed order, and writes one partial row; a
// second launch adds the partials in order.  No atomics: results are the same on every run.
//
// Everything between loads and stores is fp32; variances are of the centred values.
//
// 65536 rows of 1024, bf16, RMS norm, sigmoid gate, stream and LayerNorm: forward 142 us (4.7
// TB/s), backward 252 (4.3 TB/s); a large copy reaches 5.15.
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
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
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
    for (int i = 0; i < 4; ++i) {
      const bf16x2 h = {(__bf16)v[2 * i], (__bf16)v[2 * i + 1]};
      w[i] = __builtin_bit_cast(unsigned, h);
      asm("" : "+v"(w[i]));  // keeps the pair one packed conversion
    }
    q = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
__device__ __forceinline__ float rn_ld1(const float* p) { return *p; }
__device__ __forceinline__ float rn_ld1(const u16* p) { return __uint_as_float((unsigned)*p << 16); }
__device__ __forceinline__ void rn_st1(float* p, float x) { *p = x; }
__device__ __forceinline__ void rn_st1(u16* p, float x) { *p = __builtin_bit_cast(u16, (__bf16)x); }

// Whether element c + i of a row of D is in it.  VEC: D and every row start are multiples of 16
// bytes, so the 8 elements from c on are in the row or past it together.
template <bool VEC>
__device__ __forceinline__ bool rn_in(int c, int i, int D) {
  return VEC ? c < D : c + i < D;
}
// Elements c .. c + 7 of a row; past it they read as 0 and are not written.
template <typename E, bool VEC>
__device__ __forceinline__ void rn_load(const E* row, int c, int D, float (&v)[8]) {
  if constexpr (VEC) {
    // A load under no condition: one under it is waited for where the branches meet.
    reinterpret_cast<const Vec8<E>*>(row + (c < D ? c : 0))->get(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c < D ? v[i] : 0.f;
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
// 8 elements as they lie in memory (VEC) or widened, loaded now and looked at later.
template <typename E, bool VEC>
struct RnRaw {
  Vec8<E> q;
  __device__ __forceinline__ void load(const E* row, int c, int D) {
    q = *reinterpret_cast<const Vec8<E>*>(row + (c < D ? c : 0));
  }
  __device__ __forceinline__ void get(int c, int D, float (&v)[8]) const {
    q.get(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c < D ? v[i] : 0.f;
  }
};
template <typename E>
struct RnRaw<E, false> {
  float q[8];
  __device__ __forceinline__ void load(const E* row, int c, int D) {
    rn_load<E, false>(row, c, D, q);
  }
  __device__ __forceinline__ void get(int, int, float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = q[i];
  }
};
// Elements of a row vector, `other` where there is none.  They are read again for every row:
// the caches hold them, registers for them would cost the waves that hide the rows' loads.
template <typename P, bool VEC>
__device__ __forceinline__ void rn_vector(const void* p, float other, int c, int D, float (&v)[8]) {
  if (p) {
    asm volatile("" : "+s"(p));  // or the compiler would load it once, before the loop
    rn_load<P, VEC>((const P*)p, c, D, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = other;
  }
}

constexpr int rn_threads(int tpr) { return tpr > 256 ? tpr : 256; }

// A row's sums over its TPR lanes, in every one of them.  Past one wave the waves' sums meet
// in LDS; `turn` alternates between two sets of slots, so one barrier is enough: a wave can
// be at most one sum ahead of the others.
template <int TPR, int N>
__device__ __forceinline__ void rn_sum(float (&s)[N], int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = mg_group_sum<(TPR < MG_WAVE ? TPR : MG_WAVE)>(s[i]);
  if constexpr (TPR > MG_WAVE) {
    constexpr int W = TPR / MG_WAVE;
    __shared__ float slots[2][N][rn_threads(TPR) / MG_WAVE];
    const int w = mg_uniform(threadIdx.x / MG_WAVE), first = w / W * W;
    if ((threadIdx.x & (MG_WAVE - 1)) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) slots[turn][i][w] = s[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = 0.f;
#pragma unroll
      for (int j = 0; j < W; ++j) t += slots[turn][i][first + j];
      s[i] = t;
    }
    turn ^= 1;
  }
}

// Mean and reciprocal deviation of a row held in v (elements past D are 0).
template <int TPR, bool VEC>
__device__ __forceinline__ float2 rn_stats(const float (&v)[8], int kind, int c, int D, float eps,
                                           int& turn) {
  const float inv = 1.f / (float)D;
  float mean = 0.f;
  if (kind == RN_LAYER) {
    float s[1] = {((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]))};
    rn_sum<TPR>(s, turn);
    mean = s[0] * inv;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = v[i] - mean;
    q[0] += rn_in<VEC>(c, i, D) ? d * d : 0.f;
  }
  rn_sum<TPR>(q, turn);
  return make_float2(mean, 1.f / sqrtf(q[0] * inv + eps));
}

// 1 / (1 + e^-x) from the hardware's exponential and reciprocal, each 1 ulp off at most.  For fp32
// rows, what the product x log2 e rounds off is put back: 2e-7 of the result at any x, where it would
// be up to 6e-8 |x| (4e-6 at -87).  An infinite x leaves a NaN in the factor, which fmaxf drops.
// For bf16 rows, rounded to 2^-9, it stays off (norm-train 389 us, with it 397).
template <typename E>
__device__ __forceinline__ float rn_sigmoid(float x) {
  const float t = -1.44269502f * x;  // log2 e = 1.44269502 + 1.92596e-8
  float e = __builtin_amdgcn_exp2f(t);
  if constexpr (sizeof(E) == 4) {
    const float rest = fmaf(-1.92596299e-8f, x, fmaf(-1.44269502f, x, -t));
    e *= fmaxf(fmaf(0.693147181f, rest, 1.f), 0.5f);
  }
  return __builtin_amdgcn_rcpf(1.f + e);
}

template <typename E, typename P, int TPR, bool VEC>
__global__ __launch_bounds__(rn_threads(TPR)) void residual_norm_fwd(RnArgs a) {
  constexpr int ROWS = rn_threads(TPR) / TPR;
  const int c = (threadIdx.x % TPR) * 8, D = a.D;
  int turn = 0;
  // A group past the last row repeats it without storing, so that whole waves stay active.
  for (int64_t base = (int64_t)blockIdx.x * ROWS; base < a.rows; base += (int64_t)gridDim.x * ROWS) {
    const int64_t at = base + threadIdx.x / TPR;
    const bool live = at < a.rows;
    const int64_t row = live ? at : a.rows - 1;
    float u[8], xv[8], gv[8], w[8], b[8];
    rn_load<E, VEC>((const E*)a.h + row * a.ldh, c, D, u);
    if (a.x) rn_load<E, VEC>((const E*)a.x + row * a.ldx, c, D, xv);
    if (a.act) rn_load<E, VEC>((const E*)a.gate + row * a.ldg, c, D, gv);
    float4 st = make_float4(0.f, 1.f, 0.f, 1.f);
    if (a.post) {
      rn_vector<P, VEC>(a.post_w, 1.f, c, D, w);
      rn_vector<P, VEC>(a.post_b, 0.f, c, D, b);
      const float2 m = rn_stats<TPR, VEC>(u, a.post, c, D, a.eps, turn);
      st.x = m.x, st.y = m.y;
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = (u[i] - m.x) * m.y * w[i] + b[i];
    }
    if (a.act) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float s = rn_sigmoid<E>(gv[i]);
        u[i] *= a.act == RN_SILU ? s * gv[i] : s;
      }
    }
    if (a.x) {
      rn_vector<P, VEC>(a.scale, a.scale_const, c, D, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = xv[i] + w[i] * u[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = rn_in<VEC>(c, i, D) ? u[i] : 0.f;  // not what a bias left
    if (a.r && live) rn_store<E, VEC>((E*)a.r + row * D, c, D, u);
    if (a.pre) {
      rn_vector<P, VEC>(a.pre_w, 1.f, c, D, w);
      rn_vector<P, VEC>(a.pre_b, 0.f, c, D, b);
      const float2 m = rn_stats<TPR, VEC>(u, a.pre, c, D, a.eps, turn);
      st.z = m.x, st.w = m.y;
      if (live) {
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = (u[i] - m.x) * m.y * w[i] + b[i];
        rn_store<E, VEC>((E*)a.y + row * D, c, D, u);
      }
    }
    if (a.stats && live && threadIdx.x % TPR == 0) a.stats[row] = st;
  }
}

template <typename E, typename P, int TPR, bool VEC>
__global__ __launch_bounds__(rn_threads(TPR)) void residual_norm_bwd(RnArgs a) {
  constexpr int ROWS = rn_threads(TPR) / TPR;
  const int c = (threadIdx.x % TPR) * 8, D = a.D;
  const float inv = 1.f / (float)D;
  // A row of one element: dn (1 - n^2) would cancel down to its rounding; 1 - n^2 = eps rstd^2.
  const auto lone = [&](int kind) { return D == 1 && kind == RN_RMS; };
  float sum[RN_NPAR][8];
#pragma unroll
  for (int p = 0; p < RN_NPAR; ++p)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[p][i] = 0.f;
  int turn = 0;
  // A row's loads are issued while the row before it is worked on: the sums leave registers for
  // two or three waves a SIMD only, whose loads would otherwise come in bursts.
  struct Rows {
    RnRaw<E, VEC> h, x, g, dr, dy;
    float4 st;
  };
  const auto fetch = [&](int64_t base) {
    const int64_t at = base + threadIdx.x / TPR, row = at < a.rows ? at : a.rows - 1;
    Rows r;
    r.h.load((const E*)a.h + row * a.ldh, c, D);
    if (a.dy && a.x) r.x.load((const E*)a.x + row * a.ldx, c, D);
    if (a.act) r.g.load((const E*)a.gate + row * a.ldg, c, D);
    if (a.dr) r.dr.load((const E*)a.dr + row * a.lddr, c, D);
    if (a.dy) r.dy.load((const E*)a.dy + row * a.lddy, c, D);
    r.st = a.stats ? a.stats[row] : make_float4(0.f, 1.f, 0.f, 1.f);
    return r;
  };
  constexpr bool AHEAD = TPR < 1024;  // 16 waves have 128 registers each
  Rows next;
  if constexpr (AHEAD) next = fetch((int64_t)blockIdx.x * ROWS);
  for (int64_t base = (int64_t)blockIdx.x * ROWS; base < a.rows; base += (int64_t)gridDim.x * ROWS) {
    const int64_t row = base + threadIdx.x / TPR;
    const bool live = row < a.rows;
    const Rows now = AHEAD ? next : fetch(base);
    if constexpr (AHEAD) next = fetch(base + (int64_t)gridDim.x * ROWS);
    float n[8], xv[8], gv[8], g[8], dy[8];
    now.h.get(c, D, n);
    if (a.dy && a.x) now.x.get(c, D, xv);
    if (a.act) now.g.get(c, D, gv);
    if (a.dr) {
      now.dr.get(c, D, g);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = 0.f;
    }
    if (a.dy) now.dy.get(c, D, dy);
    const float4 st = now.st;
    // n: the post norm's rows; p = n w + b; f = act(gate), slope = act'(gate); u = p f.
    float p[8], f[8], slope[8], w[8], sc[8];
    rn_vector<P, VEC>(a.scale, a.scale_const, c, D, sc);
    if (a.post) {
      float b[8];
      rn_vector<P, VEC>(a.post_w, 1.f, c, D, w);
      rn_vector<P, VEC>(a.post_b, 0.f, c, D, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        n[i] = (n[i] - st.x) * st.y;
        p[i] = n[i] * w[i] + b[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = 1.f, p[i] = n[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[i] = 1.f, slope[i] = 0.f;
      if (a.act) {
        const float s = rn_sigmoid<E>(gv[i]), ds = s * (1.f - s);
        f[i] = a.act == RN_SILU ? s * gv[i] : s;
        slope[i] = a.act == RN_SILU ? s + gv[i] * ds : ds;
      }
    }
    if (a.dy) {
      float qw[8], s[2] = {0.f, 0.f};
      rn_vector<P, VEC>(a.pre_w, 1.f, c, D, qw);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float r = a.x ? xv[i] + sc[i] * (p[i] * f[i]) : p[i] * f[i];
        xv[i] = (r - st.z) * st.w;  // the pre norm's rows
        if (live) sum[RN_DPRE_W][i] += dy[i] * xv[i], sum[RN_DPRE_B][i] += dy[i];
        dy[i] *= qw[i];
        s[0] += dy[i] * xv[i];  // dy is 0 past D
        s[1] += dy[i];
      }
      rn_sum<TPR>(s, turn);
      const float m0 = s[0] * inv, m1 = a.pre == RN_LAYER ? s[1] * inv : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = dy[i] - xv[i] * m0 - m1;
        g[i] += st.w * (lone(a.pre) ? dy[i] * (a.eps * st.w * st.w) : d);
      }
    }
    if (a.dx && live) rn_store<E, VEC>((E*)a.dx + row * D, c, D, g);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (live) sum[RN_DSCALE][i] += g[i] * (p[i] * f[i]);
      const float du = rn_in<VEC>(c, i, D) ? (a.x ? g[i] * sc[i] : g[i]) : 0.f;
      gv[i] = du * p[i] * slope[i];
      const float dp = du * f[i];
      if (live) sum[RN_DPOST_W][i] += dp * n[i], sum[RN_DPOST_B][i] += dp;
      g[i] = dp * w[i];
      s[0] += g[i] * n[i];
      s[1] += g[i];
    }
    if (a.dgate && live) rn_store<E, VEC>((E*)a.dgate + row * D, c, D, gv);
    if (a.post) {
      rn_sum<TPR>(s, turn);
      const float m0 = s[0] * inv, m1 = a.post == RN_LAYER ? s[1] * inv : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = g[i] - n[i] * m0 - m1;
        g[i] = st.y * (lone(a.post) ? g[i] * (a.eps * st.y * st.y) : d);
      }
    }
    if (a.dh && live) rn_store<E, VEC>((E*)a.dh + row * D, c, D, g);
  }
  if (!a.part) return;
  // Over the workgroup's groups, then one partial row for each workgroup.
  float* part = a.part + (int64_t)blockIdx.x * RN_NPAR * D;
  if constexpr (ROWS == 1) {
#pragma unroll
    for (int p = 0; p < RN_NPAR; ++p)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < D) part[p * D + c + i] = sum[p][i];
  } else {
    __shared__ float s[ROWS][TPR * 8 + 4];
#pragma unroll
    for (int p = 0; p < RN_NPAR; ++p) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) s[threadIdx.x / TPR][c + i] = sum[p][i];
      __syncthreads();
      for (int x = threadIdx.x; x < TPR * 8 && x < D; x += rn_threads(TPR)) {
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < ROWS; ++j) t += s[j][x];
        part[p * D + x] = t;
      }
    }
  }
}

struct RnOut {
  void* p[RN_NPAR];
};

// out[c] = sum over the partial rows, in a fixed order: 16 waves take every sixteenth row of 64
// columns.
constexpr int RN_SUM_WAVES = 16;
template <typename P>
__global__ __launch_bounds__(RN_SUM_WAVES* MG_WAVE) void residual_norm_sums(
    const float* __restrict__ part, RnOut out, int parts, int D) {
  __shared__ float s[RN_SUM_WAVES][MG_WAVE];
  const int lane = threadIdx.x & (MG_WAVE - 1), w = threadIdx.x / MG_WAVE;
  P* dst = (P*)out.p[blockIdx.y];
  if (!dst) return;
  const int col = blockIdx.x * MG_WAVE + lane, c = col < D ? col : D - 1;
  const float* src = part + (int64_t)blockIdx.y * D + c;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  int r = w;
  for (; r + 3 * RN_SUM_WAVES < parts; r += 4 * RN_SUM_WAVES) {
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] += src[(int64_t)(r + RN_SUM_WAVES * i) * RN_NPAR * D];
  }
  for (; r < parts; r += RN_SUM_WAVES) a[0] += src[(int64_t)r * RN_NPAR * D];
  s[w][lane] = (a[0] + a[1]) + (a[2] + a[3]);
  __syncthreads();
  if (w != 0 || col >= D) return;
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < RN_SUM_WAVES; ++i) t += s[i][lane];
  rn_st1(dst + col, t);
}

// A row's lanes: the fewest that hold it with 8 elements each, so that narrow rows share a wave
// and a wide one has a workgroup.  (Wider rows at 16 elements a lane had one wave a SIMD in the
// backward, 256 registers: 65536 rows of 1024 in bf16 took 670 us, at 8 elements a lane 397, and
// with a row's loads a row ahead 258.)
int rn_tpr(int64_t D) {
  int n = 16;
  while (n * 8 < D) n *= 2;
  return n;
}

// Workgroups: enough to fill the chip several times over; each has partial sums to write, so
// the backward takes no more than RN_PARTS.
constexpr int64_t RN_GRID = 8192, RN_PARTS = 512;
int64_t rn_grid(int64_t rows, int64_t D, int64_t most) {
  const int tpr = rn_tpr(D), per = tpr > 256 ? 1 : 256 / tpr;
  const int64_t n = (rows + per - 1) / per;
  return n < most ? n : most;
}

bool rn_ok(int64_t rows, int64_t D) { return rows >= 1 && D >= 1 && D <= 8192 && rows <= (1ll << 40) / D; }

bool rn_vec(const void* p, int64_t ld, int esize) {
  return !p || (((uintptr_t)p & 15) == 0 && (ld * esize) % 16 == 0);
}

template <typename E, typename P, int TPR, bool VEC>
void rn_launch(const RnArgs& a, bool bwd, unsigned grid, hipStream_t stream) {
  const dim3 nt(rn_threads(TPR));
  if (bwd)
    hipLaunchKernelGGL((residual_norm_bwd<E, P, TPR, VEC>), dim3(grid), nt, 0, stream, a);
  else
    hipLaunchKernelGGL((residual_norm_fwd<E, P, TPR, VEC>), dim3(grid), nt, 0, stream, a);
}
template <typename E, typename P, int TPR>
void rn_pick(const RnArgs& a, bool vec, bool bwd, unsigned grid, hipStream_t stream) {
  if (vec) rn_launch<E, P, TPR, true>(a, bwd, grid, stream);
  else rn_launch<E, P, TPR, false>(a, bwd, grid, stream);
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
    case 32: rn_pick<E, P, 32>(a, vec, bwd, grid, stream); break;
    case 64: rn_pick<E, P, 64>(a, vec, bwd, grid, stream); break;
    case 128: rn_pick<E, P, 128>(a, vec, bwd, grid, stream); break;
    case 256: rn_pick<E, P, 256>(a, vec, bwd, grid, stream); break;
    case 512: rn_pick<E, P, 512>(a, vec, bwd, grid, stream); break;
    default: rn_pick<E, P, 1024>(a, vec, bwd, grid, stream);
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
    hipLaunchKernelGGL(residual_norm_sums<u16>, g, dim3(RN_SUM_WAVES * MG_WAVE), 0, stream, a.part, out, (int)grid,
                       (int)D);
  else
    hipLaunchKernelGGL(residual_norm_sums<float>, g, dim3(RN_SUM_WAVES * MG_WAVE), 0, stream, a.part, out, (int)grid,
                       (int)D);
  return hipGetLastError() == hipSuccess ? MG_OK : MG_ERR_LAUNCH;
}

}  // extern "C"
