// Linear attention with a decay for each head (gfx950).
//
//   S_t = a_t S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t,   a_t = exp(g_t)
//
// per batch and head, S (dk, dv) in fp32.  In chunks of C tokens, with G_i = g_1 + ... + g_i
// of the chunk, D_ij = exp(G_i - G_j) for j <= i, S the state before the chunk and R the
// adjoint of the state after it:
//
//   o_i  = scale (e^{G_i} S^T q_i + sum_{j<=i} D_ij (q_i.k_j) v_j)
//   S'   = e^{G_C} S + sum_j (D_Cj k_j) v_j^T
//   dq_i = scale (e^{G_i} S do_i + sum_{j<=i} D_ij (do_i.v_j) k_j)
//   dk_j = D_Cj R v_j   + scale sum_{i>=j} D_ij (do_i.v_j) q_i
//   dv_j = D_Cj R^T k_j + scale sum_{i>=j} D_ij (q_i.k_j) do_i
//   R'   = e^{G_C} R + sum_i (scale e^{G_i} q_i) do_i^T
//
// Every exponent is a sum over a span of the chunk, so nothing overflows for g <= 0 and
// nothing is divided.  The sums G are formed in fp64 and kept as two floats: near pairs deep
// in a chunk are differences of large sums.  A step whose factor is below the smallest normal
// float (-inf among them) starts over: steps before and after it are told apart by a count,
// which keeps the sums finite.
//
// Gradient of g.  G_i enters o_i with do_i.o_i and every later use of k_j v_j^T with -k_j.dk_j:
//   e_i = sum_{j<i} X_ij - sum_{j>i} X_ji + q_i.dq_i^inter - k_i.dk_i^inter,
//   X_ij = scale D_ij (q_i.k_j)(do_i.v_j),
// the diagonal cancelling exactly, and dg_t = sum_{i>=t} e_i + <R_end, S_end> over a segment,
// so that what cancels in the sum is never longer than a segment.
//
// Split.  A workgroup of 8 waves walks over the chunks of one (batch, head, segment) with the
// state in its registers (32 a lane at dk = dv = 128): the state never goes through memory
// except at the segments' ends.  Where there are fewer (batch, head) pairs than the chip
// holds workgroups, a sequence is cut into segments: a first pass forms each segment's own
// contribution, a scan joins them, and the main pass starts every segment from its state.
//
// Products run on the matrix cores, 16 x 16 tiles: bf16 inputs with
// v_mfma_f32_16x16x32_bf16, fp32 inputs with v_mfma_f32_16x16x4_f32 (C = 32).  Operands lie
// in LDS as they lie in memory, (token, feature) and (dk, dv); where the contracted index is
// the slow one a bf16 fragment comes from two ds_read_b64_tr_b16.  Rounding, bf16: inputs are
// exact.  What only feeds bf16 outputs (the C x C matrices, the state in o and dv) is rounded
// to bf16 once; what feeds fp32 outputs (decayed keys and queries into the states, the states
// into the gradient of g) is held as hi + lo, 16 significant bits, at twice the products.
//
// Bound: LDS reads of operand fragments, then memory.
#include "mg_common.h"

namespace {

typedef uint16_t u16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int NT = 512, NW = NT / MG_WAVE;

enum { LA_STATE = 0, LA_OUT = 1, LA_RSTATE = 2, LA_DQ = 3, LA_DKV = 4 };

struct LaArgs {
  const void *q, *k, *v, *dout;
  const float* g;
  const int* lengths;
  // strides in elements: batch, token, head
  int64_t qs[3], ks[3], vs[3], ds[3], gs[3];
  int64_t T;
  int H, group, dk, dv;  // heads of v, v heads for each key head
  float scale;
  int segs, per;        // segments of a sequence, chunks of a segment
  const float* first;   // (BH, dk, dv) state before the first segment, or null for zero
  float* last;          // (BH, dk, dv) state after the last one, or null
  float* bound;         // (BH, segs - 1, dk, dv): what LA_STATE adds, then states between segments
  float* decay;         // (BH, segs - 1)
  void *out, *out2;     // o; dq; dk and dv
  float *part;          // (B, T, H, dk) fp32 in place of out where heads share it
  float* e;             // (BH, T)
};

// ---- operands ------------------------------------------------------------------------
template <typename T>
struct Op;

template <>
struct Op<u16> {
  typedef bf16x8 Frag;
  static constexpr int KB = 32, VE = 8, PAD = 8, PLANES = 2;
  // Rows of the free index, the contracted one consecutive.
  static __device__ __forceinline__ Frag near(const u16* m, int ld, int r0, int k0) {
    const int l = threadIdx.x & 63;
    return *reinterpret_cast<const bf16x8*>(m + (r0 + (l & 15)) * ld + k0 + 8 * (l >> 4));
  }
  // Rows of the contracted index: 16 lanes fetch 4 rows x 16 columns and get a column each.
  static __device__ __forceinline__ Frag far(const u16* m, int ld, int c0, int k0) {
    const int l = threadIdx.x & 63;
    const u16* p = m + (k0 + 8 * (l >> 4) + ((l & 15) >> 2)) * ld + c0 + 4 * (l & 3);
    typedef __attribute__((address_space(3))) s16x4* lds_t;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)p);
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(p + 4 * ld));
    const s16x8 x = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return __builtin_bit_cast(bf16x8, x);
  }
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

template <>
struct Op<float> {
  typedef f32x4 Frag;
  static constexpr int KB = 16, VE = 4, PAD = 4, PLANES = 1;
  static __device__ __forceinline__ Frag near(const float* m, int ld, int r0, int k0) {
    const int l = threadIdx.x & 63;
    return *reinterpret_cast<const f32x4*>(m + (r0 + (l & 15)) * ld + k0 + 4 * (l >> 4));
  }
  static __device__ __forceinline__ Frag far(const float* m, int ld, int c0, int k0) {
    const int l = threadIdx.x & 63;
    const float* p = m + (k0 + 4 * (l >> 4)) * ld + c0 + (l & 15);
    const f32x4 x = {p[0], p[ld], p[2 * ld], p[3 * ld]};
    return x;
  }
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

// The wave's tiles of an Mt x Nt grid of 16 x 16 tiles over 8 waves, WM of them along M.
template <int Mt, int Nt, int WM_>
struct Tiling {
  static constexpr int WM = Mt < WM_ ? Mt : WM_, WN = NW / WM;
  static constexpr int TM = Mt / WM, TN = Nt < WN ? 1 : Nt / WN;
  static_assert(Mt % WM == 0 && (Nt < WN || Nt % WN == 0), "tiles divide among the waves");
  static __device__ __forceinline__ int wm() { return mg_uniform(threadIdx.x >> 6) % WM; }
  static __device__ __forceinline__ int wn() { return mg_uniform(threadIdx.x >> 6) / WM; }
  static __device__ __forceinline__ bool live() { return Nt >= WN || wn() < Nt; }
  static __device__ __forceinline__ int m0(int t) { return 16 * (wm() * TM + t); }
  static __device__ __forceinline__ int n0(int t) { return 16 * (wn() * TN + t); }
};

// acc[tm][tn] += A B over K contracted elements: A (free index M) and B (free index N) each
// near or far, in AP and BP planes of hi and lo (their lo lo product is below fp32's rounding
// of the sum and left out).
template <typename T, typename Ti, int K, bool AFAR, bool BFAR, int AP, int BP>
__device__ __forceinline__ void product(f32x4 (&acc)[Ti::TM][Ti::TN], const T* A, int lda, int pa,
                                        const T* B, int ldb, int pb) {
  if (!Ti::live()) return;
#pragma unroll
  for (int k0 = 0; k0 < K; k0 += Op<T>::KB) {
    typename Op<T>::Frag a[AP][Ti::TM], b[BP][Ti::TN];
#pragma unroll
    for (int p = 0; p < AP; ++p)
#pragma unroll
      for (int t = 0; t < Ti::TM; ++t)
        a[p][t] = AFAR ? Op<T>::far(A + p * pa, lda, Ti::m0(t), k0)
                       : Op<T>::near(A + p * pa, lda, Ti::m0(t), k0);
#pragma unroll
    for (int p = 0; p < BP; ++p)
#pragma unroll
      for (int t = 0; t < Ti::TN; ++t)
        b[p][t] = BFAR ? Op<T>::far(B + p * pb, ldb, Ti::n0(t), k0)
                       : Op<T>::near(B + p * pb, ldb, Ti::n0(t), k0);
#pragma unroll
    for (int i = 0; i < Ti::TM; ++i)
#pragma unroll
      for (int j = 0; j < Ti::TN; ++j) {
        acc[i][j] = Op<T>::mma(a[0][i], b[0][j], acc[i][j]);
        if constexpr (AP > 1) acc[i][j] = Op<T>::mma(a[1][i], b[0][j], acc[i][j]);
        if constexpr (BP > 1) acc[i][j] = Op<T>::mma(a[0][i], b[1][j], acc[i][j]);
      }
  }
}

template <typename Ti>
__device__ __forceinline__ void clear(f32x4 (&acc)[Ti::TM][Ti::TN]) {
#pragma unroll
  for (int i = 0; i < Ti::TM; ++i)
#pragma unroll
    for (int j = 0; j < Ti::TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// ---- elements --------------------------------------------------------------------------
__device__ __forceinline__ float to_f(u16 x) { return __uint_as_float((unsigned)x << 16); }
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ unsigned pack2(float x, float y) {
  const bf16x2 h = {(__bf16)x, (__bf16)y};
  return __builtin_bit_cast(unsigned, h);
}
// x = hi + lo, both rounded to nearest, two values at a time.
__device__ __forceinline__ void split2(float x, float y, unsigned& hi, unsigned& lo) {
  hi = pack2(x, y);
  lo = pack2(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
}

// Four consecutive elements into LDS, in PL planes `plane` elements apart.
template <int PL>
__device__ __forceinline__ void put4(u16* p, int plane, f32x4 x) {
  if constexpr (PL == 2) {
    unsigned h0, l0, h1, l1;
    split2(x[0], x[1], h0, l0);
    split2(x[2], x[3], h1, l1);
    *reinterpret_cast<uint2*>(p) = make_uint2(h0, h1);
    *reinterpret_cast<uint2*>(p + plane) = make_uint2(l0, l1);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2(x[0], x[1]), pack2(x[2], x[3]));
  }
}
template <int PL>
__device__ __forceinline__ void put4(float* p, int, f32x4 x) {
  *reinterpret_cast<f32x4*>(p) = x;
}

// Four consecutive elements from column c of a row of d, to memory.
__device__ __forceinline__ void store4(u16* p, int c, int d, f32x4 x) {
  if (c + 4 <= d && (((uintptr_t)(p + c)) & 7) == 0) {
    *reinterpret_cast<uint2*>(p + c) = make_uint2(pack2(x[0], x[1]), pack2(x[2], x[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < d) p[c + i] = __builtin_bit_cast(u16, (__bf16)x[i]);
  }
}
__device__ __forceinline__ void store4(float* p, int c, int d, f32x4 x) {
  if (c + 4 <= d && (((uintptr_t)(p + c)) & 15) == 0) {
    *reinterpret_cast<f32x4*>(p + c) = x;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < d) p[c + i] = x[i];
  }
}

// A chunk's (C, D) block on its way from memory to LDS, 16 bytes a vector; 0 outside the
// sequence and the d columns.
template <typename T, int C, int D>
struct Block {
  static constexpr int VE = Op<T>::VE, N = C * D / VE / NT, LD = D + Op<T>::PAD;
  static_assert(C * D % (VE * NT) == 0, "whole vectors for every thread");
  uint4 x[N];

  static __device__ __forceinline__ int row(int n) { return (threadIdx.x + n * NT) / (D / VE); }
  static __device__ __forceinline__ int col(int n) {
    return (threadIdx.x + n * NT) % (D / VE) * VE;
  }
  // src: the chunk's first row; ld: elements between rows; wide: 16-byte vectors are aligned
  // and lie inside the row or outside it.
  __device__ __forceinline__ void load(const T* src, int64_t ld, int rows, int d, bool wide) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      x[n] = make_uint4(0u, 0u, 0u, 0u);
      const int r = row(n), c = col(n);
      if (r >= rows) continue;
      const T* p = src + r * ld + c;
      if (wide) {
        if (c < d) x[n] = *reinterpret_cast<const uint4*>(p);
      } else {
        T e[VE];
#pragma unroll
        for (int i = 0; i < VE; ++i) e[i] = c + i < d ? p[i] : (T)0;
        __builtin_memcpy(&x[n], e, 16);
      }
    }
  }
  __device__ __forceinline__ void put(T* m) const {
#pragma unroll
    for (int n = 0; n < N; ++n) *reinterpret_cast<uint4*>(m + row(n) * LD + col(n)) = x[n];
  }
  __device__ __forceinline__ void get(const T* m) {
#pragma unroll
    for (int n = 0; n < N; ++n) x[n] = *reinterpret_cast<const uint4*>(m + row(n) * LD + col(n));
  }
  // Rows times w[row], in all planes.
  __device__ __forceinline__ void put_scaled(T* m, const float* w) const {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const float s = w[row(n)];
      T e[VE];
      __builtin_memcpy(e, &x[n], 16);
#pragma unroll
      for (int i = 0; i < VE; i += 4) {
        const f32x4 y = {s * to_f(e[i]), s * to_f(e[i + 1]), s * to_f(e[i + 2]),
                         s * to_f(e[i + 3])};
        put4<Op<T>::PLANES>(m + row(n) * LD + col(n) + i, C * LD, y);
      }
    }
  }
};

// ---- decays ------------------------------------------------------------------------------
// G_i as hi + lo in powers of two, and the count of steps that start over up to i.
struct Gate {
  float hi, lo, n, pad;
};
__device__ __forceinline__ float span(const Gate& i, const Gate& j) {  // exp(G_i - G_j)
  return __builtin_amdgcn_exp2f(fmaf(-1e6f, i.n - j.n, (i.hi - j.hi) + (i.lo - j.lo)));
}
__device__ __forceinline__ float span0(const Gate& i) {
  return __builtin_amdgcn_exp2f(fmaf(-1e6f, i.n, i.hi + i.lo));
}

// One wave: lane i forms the chunk's i-th gate from its g (0 past the sequence).
template <int C>
__device__ __forceinline__ void make_gates(Gate* out, float g) {
  const int l = threadIdx.x & 63;
  constexpr double LOG2E = 1.4426950408889634;
  double s = (double)g * LOG2E;
  const bool over = s < -126.0;
  float n = over ? 1.f : 0.f;
  s = over ? 0.0 : s;
#pragma unroll
  for (int d = 1; d < C; d *= 2) {
    const double t = __shfl_up(s, d);
    const float u = __shfl_up(n, d);
    if (l >= d) s += t, n += u;
  }
  const float hi = (float)s;
  if (l < C) out[l] = Gate{hi, (float)(s - (double)hi), n, 0.f};
}

// ---- the sweep -------------------------------------------------------------------------------
template <typename T, int C, int DK, int DV, int MODE>
struct Lds {
  static constexpr int E = sizeof(T), PAD = Op<T>::PAD, PL = Op<T>::PLANES;
  static constexpr int LK = DK + PAD, LV = DV + PAD, LC = C + PAD;
  static constexpr bool GRAD = MODE == LA_DQ || MODE == LA_DKV;
  static constexpr bool BARE = MODE == LA_STATE || MODE == LA_RSTATE;
  static constexpr int Q = 0;  // queries
  static constexpr int K = Q + (BARE ? 0 : C * LK);
  static constexpr int V = K + (BARE ? 0 : C * LK);
  static constexpr int O = V + C * LV;  // output gradients
  static constexpr int P = O + (GRAD ? C * LV : 0);
  static constexpr int P2 = P + (BARE ? 0 : C * LC);
  static constexpr int S = P2 + (MODE == LA_DKV ? C * LC : 0);  // state
  static constexpr int SPLANES = GRAD ? PL : 1;
  static constexpr int SSIZE = BARE ? 0 : DK * LV * SPLANES;
  // decayed keys (queries): in the state's place where it has been read by then
  static constexpr int W = GRAD ? S : S + SSIZE;
  static constexpr int WSIZE = C * LK * PL;
  static constexpr int END = GRAD ? S + (SSIZE > WSIZE ? SSIZE : WSIZE) : W + WSIZE;
  static constexpr int BYTES = (END * E + 15) / 16 * 16;
};

template <typename T, int C, int DK, int DV, int MODE>
__global__ __launch_bounds__(NT, 2) void la_sweep(LaArgs a) {
  typedef Lds<T, C, DK, DV, MODE> L;
  constexpr int PL = L::PL, LK = L::LK, LV = L::LV, LC = L::LC;
  constexpr bool REV = MODE == LA_RSTATE || MODE == LA_DKV, BARE = L::BARE, GRAD = L::GRAD;
  typedef Tiling<DV / 16, DK / 16, 2> TS;  // the state, transposed: M = dv, N = dk
  typedef Tiling<C / 16, C / 16, 4> TC;    // chunk matrices
  typedef Tiling<DK / 16, C / 16, 4> TK;   // (dk, token)
  typedef Tiling<DV / 16, C / 16, 4> TV;   // (dv, token)
  __shared__ __align__(16) char raw[L::BYTES];
  __shared__ Gate gates[2][C];
  __shared__ float s_w[C];
  // Sums over the chunk matrices' rows and columns, and rows' products with dq or dk, by wave.
  __shared__ float s_row[4][C], s_col[4][C], s_dot[4][C];
  T* lds = reinterpret_cast<T*>(raw);
  T *sQ = lds + L::Q, *sK = lds + L::K, *sV = lds + L::V, *sO = lds + L::O, *sP = lds + L::P,
    *sP2 = lds + L::P2, *sS = lds + L::S, *sW = lds + L::W;

  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = mg_uniform(tid >> 6);
  const int64_t bh = blockIdx.x;
  const int seg = blockIdx.y;  // bare passes: the last (first) segment's state isn't needed
  const int b = (int)(bh / a.H), h = (int)(bh % a.H), kh = h / a.group;
  const int dk = a.dk, dv = a.dv;
  const int64_t T_ = a.T;
  int64_t len = T_;
  if (a.lengths) {
    const int64_t n = a.lengths[b];
    len = n < 0 ? 0 : n < T_ ? n : T_;
  }
  const int s_at = MODE == LA_RSTATE ? seg + 1 : seg;
  const int64_t t0 = (int64_t)s_at * a.per * C;                       // the segment's tokens
  const int64_t t1 = t0 + (int64_t)a.per * C < T_ ? t0 + (int64_t)a.per * C : T_;
  const int64_t e1 = len < t1 ? len : t1;                               // and its live ones' end
  const int chunks = e1 > t0 ? (int)((e1 - t0 + C - 1) / C) : 0;

  const T* q = (const T*)a.q + b * a.qs[0] + kh * a.qs[2];
  const T* k = (const T*)a.k + b * a.ks[0] + kh * a.ks[2];
  const T* v = (const T*)a.v + b * a.vs[0] + h * a.vs[2];
  const T* dout = (const T*)a.dout + b * a.ds[0] + h * a.ds[2];
  const float* g = a.g + b * a.gs[0] + h * a.gs[2];
  const auto wide = [&](const void* p, const int64_t (&s)[3], int d) {
    constexpr int VE = Op<T>::VE;
    return (((uintptr_t)p) & 15) == 0 && d % VE == 0 && s[0] % VE == 0 && s[1] % VE == 0 &&
           s[2] % VE == 0;
  };
  const bool wq = MODE == LA_STATE || wide(a.q, a.qs, dk), wk = wide(a.k, a.ks, dk),
             wv = wide(a.v, a.vs, dv), wo = wide(a.dout, a.ds, dv);

  // The state: lane (lg, lr) of tile (i, j) holds S[n0 + lr][m0 + 4 lg .. + 3].
  f32x4 S[TS::TM][TS::TN];
  clear<TS>(S);
  const int64_t ss = (int64_t)dk * dv;
  const auto each_state = [&](auto&& f) {
#pragma unroll
    for (int i = 0; i < TS::TM; ++i)
#pragma unroll
      for (int j = 0; j < TS::TN; ++j) f(S[i][j], TS::n0(j) + lr, TS::m0(i) + 4 * lg);
  };
  if constexpr (!BARE) {
    const float* from;
    if constexpr (REV)
      from = seg == a.segs - 1 ? (a.first ? a.first + bh * ss : nullptr)
                               : a.bound + (bh * (a.segs - 1) + seg) * ss;
    else
      from = seg == 0 ? (a.first ? a.first + bh * ss : nullptr)
                      : a.bound + (bh * (a.segs - 1) + seg - 1) * ss;
    if (from)
      each_state([&](f32x4& x, int r, int c) {
        if (r < dk) {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = c + i < dv ? from[(int64_t)r * dv + c + i] : 0.f;
        }
      });
  }

  Block<T, C, DK> bq, bk;
  Block<T, C, DV> bv, bo;
  const auto at = [&](int n) { return t0 + (int64_t)(REV ? chunks - 1 - n : n) * C; };
  const auto rows_at = [&](int64_t t) { return (int)(e1 - t < C ? e1 - t : C); };
  const auto fetch = [&](int64_t t) {
    const int rows = rows_at(t);
    if constexpr (MODE != LA_STATE) bq.load(q + t * a.qs[1], a.qs[1], rows, dk, wq);
    if constexpr (MODE != LA_RSTATE) bk.load(k + t * a.ks[1], a.ks[1], rows, dk, wk);
    if constexpr (MODE != LA_RSTATE) bv.load(v + t * a.vs[1], a.vs[1], rows, dv, wv);
    if constexpr (GRAD || MODE == LA_RSTATE) bo.load(dout + t * a.ds[1], a.ds[1], rows, dv, wo);
  };
  const auto gates_of = [&](int n) {
    const int64_t t = at(n);
    make_gates<C>(gates[n & 1], lane < rows_at(t) ? g[(t + lane) * a.gs[1]] : 0.f);
  };
  if (chunks > 0) {
    fetch(at(0));
    if (wave == 0) gates_of(0);
  }
  float fall = 1.f;  // the segment's decay so far

  for (int n = 0; n < chunks; ++n) {
    const int64_t t = at(n);
    const int rows = rows_at(t);
    const Gate* ga = gates[n & 1];
    __syncthreads();  // the gates; and the last chunk's operands are read
    if constexpr (!BARE) {
      bq.put(sQ);
      bk.put(sK);
      if constexpr (GRAD) bo.put(sO);
      each_state([&](f32x4& x, int r, int c) { put4<L::SPLANES>(sS + r * LV + c, DK * LV, x); });
    }
    const Gate end = ga[C - 1];
    const float keep = span0(end);
    if (tid < C) s_w[tid] = REV ? a.scale * span0(ga[tid]) : span(end, ga[tid]);
    if constexpr (MODE == LA_RSTATE) bo.put(sV);
    else bv.put(sV);
    if constexpr (!GRAD) {
      __syncthreads();  // s_w
      if constexpr (MODE == LA_RSTATE) bq.put_scaled(sW, s_w);
      else bk.put_scaled(sW, s_w);
    }
    __syncthreads();
    if (n + 1 < chunks) {
      fetch(at(n + 1));
      if (wave == 0) gates_of(n + 1);
    }

    if constexpr (!BARE) {
      // Chunk matrices, M the token that is contracted next, N the other: (j, i) towards the
      // queries' side, (i, j) towards the keys'.
      f32x4 A[TC::TM][TC::TN], B[TC::TM][TC::TN];
      clear<TC>(A);
      clear<TC>(B);
      if constexpr (REV) {
        product<T, TC, DK, false, false, 1, 1>(A, sQ, LK, 0, sK, LK, 0);
        product<T, TC, DV, false, false, 1, 1>(B, sO, LV, 0, sV, LV, 0);
      } else {
        product<T, TC, DK, false, false, 1, 1>(A, sK, LK, 0, sQ, LK, 0);
        if constexpr (GRAD) product<T, TC, DV, false, false, 1, 1>(B, sV, LV, 0, sO, LV, 0);
      }
      if (TC::live()) {
        float col[TC::TM][4];
#pragma unroll
        for (int im = 0; im < TC::TM; ++im)
#pragma unroll
          for (int x = 0; x < 4; ++x) col[im][x] = 0.f;
#pragma unroll
        for (int jn = 0; jn < TC::TN; ++jn) {
          const int nn = TC::n0(jn) + lr;
          const Gate gn = ga[nn];
          float row = 0.f;
#pragma unroll
          for (int im = 0; im < TC::TM; ++im) {
            const int mm = TC::m0(im) + 4 * lg;
            f32x4 p, p2;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int i = REV ? mm + x : nn, j = REV ? nn : mm + x;
              const float d = j <= i ? a.scale * (REV ? span(ga[mm + x], gn) : span(gn, ga[mm + x]))
                                     : 0.f;
              const float pa = A[im][jn][x] * d, pb = B[im][jn][x] * d;
              p[x] = MODE == LA_DQ ? pb : pa;
              p2[x] = pb;
              if constexpr (MODE == LA_DQ) {
                const float xs = j < i ? A[im][jn][x] * pb : 0.f;
                row += xs;
                col[im][x] += xs;
              }
            }
            put4<1>(sP + nn * LC + mm, 0, p);
            if constexpr (MODE == LA_DKV) put4<1>(sP2 + nn * LC + mm, 0, p2);
          }
          if constexpr (MODE == LA_DQ) {
            row = mg_pair_sum<32>(mg_pair_sum<16>(row));
            if (lane < 16) s_row[TC::wm()][nn] = row;
          }
        }
        if constexpr (MODE == LA_DQ) {
#pragma unroll
          for (int im = 0; im < TC::TM; ++im)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float s = mg_group_sum<16>(col[im][x]);
              if (lr == 0) s_col[TC::wn()][TC::m0(im) + 4 * lg + x] = s;
            }
        }
      }
      __syncthreads();
    }

    if constexpr (MODE == LA_OUT) {
      f32x4 in[TV::TM][TV::TN], ac[TV::TM][TV::TN];
      clear<TV>(in);
      clear<TV>(ac);
      product<T, TV, DK, true, false, 1, 1>(ac, sS, LV, 0, sQ, LK, 0);
      product<T, TV, C, true, false, 1, 1>(in, sV, LV, 0, sP, LC, 0);
      if (TV::live()) {
#pragma unroll
        for (int j = 0; j < TV::TN; ++j) {
          const int i = TV::n0(j) + lr;
          const float f = a.scale * span0(ga[i]);
          if (i < rows) {
            T* o = (T*)a.out + ((b * T_ + t + i) * a.H + h) * (int64_t)dv;
#pragma unroll
            for (int m = 0; m < TV::TM; ++m)
              store4(o, TV::m0(m) + 4 * lg, dv, in[m][j] + f * ac[m][j]);
          }
        }
      }
    }
    if constexpr (GRAD) {
      // dq or dk: the part through the state, then the chunk's own.
      f32x4 in[TK::TM][TK::TN], ac[TK::TM][TK::TN];
      clear<TK>(in);
      clear<TK>(ac);
      product<T, TK, DV, false, false, PL, 1>(ac, sS, LV, DK * LV, REV ? sV : sO, LV, 0);
      product<T, TK, C, true, false, 1, 1>(in, REV ? sQ : sK, LK, 0, REV ? sP2 : sP, LC, 0);
      if (TK::live()) {
#pragma unroll
        for (int j = 0; j < TK::TN; ++j) {
          const int i = TK::n0(j) + lr;
          const float f = REV ? span(end, ga[i]) : a.scale * span0(ga[i]);
          const T* x = (REV ? sK : sQ) + i * LK;
          const int64_t row = ((b * T_ + t + i) * a.H + h) * (int64_t)dk;
          float dot = 0.f;
#pragma unroll
          for (int m = 0; m < TK::TM; ++m) {
            const int c = TK::m0(m) + 4 * lg;
            const f32x4 y = f * ac[m][j];
#pragma unroll
            for (int u = 0; u < 4; ++u) dot += y[u] * to_f(x[c + u]);
            if (i < rows) {
              if (a.part) store4(a.part + row, c, dk, y + in[m][j]);
              else store4((T*)a.out + row, c, dk, y + in[m][j]);
            }
          }
          dot = mg_pair_sum<32>(mg_pair_sum<16>(dot));
          if (lane < 16) s_dot[TK::wm()][i] = dot;
        }
      }
    }
    if constexpr (MODE == LA_DKV) {
      f32x4 in[TV::TM][TV::TN], ac[TV::TM][TV::TN];
      clear<TV>(in);
      clear<TV>(ac);
      product<T, TV, DK, true, false, 1, 1>(ac, sS, LV, 0, sK, LK, 0);
      product<T, TV, C, true, false, 1, 1>(in, sO, LV, 0, sP, LC, 0);
      if (TV::live()) {
#pragma unroll
        for (int j = 0; j < TV::TN; ++j) {
          const int i = TV::n0(j) + lr;
          const float f = span(end, ga[i]);
          if (i < rows) {
            T* o = (T*)a.out2 + ((b * T_ + t + i) * a.H + h) * (int64_t)dv;
#pragma unroll
            for (int m = 0; m < TV::TM; ++m)
              store4(o, TV::m0(m) + 4 * lg, dv, in[m][j] + f * ac[m][j]);
          }
        }
      }
    }
    if constexpr (GRAD) {
      __syncthreads();  // the state's copy is read, the sums are written
      if (tid < rows) {
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < TK::WM; ++w) x += s_dot[w][tid];
        float* e = a.e + bh * T_ + t + tid;
        if constexpr (MODE == LA_DQ) {
#pragma unroll
          for (int w = 0; w < TC::WM; ++w) x += s_row[w][tid];
#pragma unroll
          for (int w = 0; w < TC::WN && w < C / 16; ++w) x -= s_col[w][tid];
          *e = x;
        } else {
          *e -= x;
        }
      }
      Block<T, C, DK> w;
      w.get(REV ? sQ : sK);
      w.put_scaled(sW, s_w);
      __syncthreads();
    }
    // The state: its decay, then the chunk's own.
#pragma unroll
    for (int i = 0; i < TS::TM; ++i)
#pragma unroll
      for (int j = 0; j < TS::TN; ++j) S[i][j] *= keep;
    product<T, TS, C, true, true, 1, PL>(S, MODE == LA_DKV ? sO : sV, LV, 0, sW, LK, C * LK);
    fall *= keep;
  }

  float* to = nullptr;
  if constexpr (BARE) {
    to = a.bound + (bh * (a.segs - 1) + seg) * ss;
    if (tid == 0) a.decay[bh * (a.segs - 1) + seg] = fall;
  } else if (seg == (REV ? 0 : a.segs - 1)) {
    to = a.last ? a.last + bh * ss : nullptr;
  }
  if (to)
    each_state([&](f32x4& x, int r, int c) {
      if (r < dk) store4(to + (int64_t)r * dv, c, dv, x);
    });
  // Past a sequence's length.
  if constexpr (!BARE) {
    const int64_t z0 = e1 > t0 ? e1 : t0;
    const auto zero = [&](auto* p, int d) {
      for (int64_t x = tid; x < (t1 - z0) * d; x += NT)
        p[((b * T_ + z0 + x / d) * a.H + h) * (int64_t)d + x % d] = 0;
    };
    if constexpr (MODE == LA_OUT) zero((T*)a.out, dv);
    if constexpr (GRAD) {
      if (a.part) zero(a.part, dk);
      else zero((T*)a.out, dk);
    }
    if constexpr (MODE == LA_DKV) zero((T*)a.out2, dv);
    if constexpr (MODE == LA_DQ)
      for (int64_t x = z0 + tid; x < t1; x += NT) a.e[bh * T_ + x] = 0.f;
  }
}

// ---- between the segments -----------------------------------------------------------------
// bound[s]: what segment s (reverse: s + 1) adds -> the state (adjoint) between s and s + 1.
__global__ __launch_bounds__(256) void la_join(const float* __restrict__ first,
                                               float* __restrict__ bound,
                                               const float* __restrict__ decay, int64_t BH,
                                               int64_t ss, int n, int rev) {
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (x >= BH * ss) return;
  const int64_t bh = x / ss, at = x % ss;
  float s = first ? first[x] : 0.f;
  for (int i = 0; i < n; ++i) {
    const int64_t seg = bh * n + (rev ? n - 1 - i : i);
    s = decay[seg] * s + bound[seg * ss + at];
    bound[seg * ss + at] = s;
  }
}

// dg_t = sum of e from t to its segment's end + <R, S> there; 0 past a sequence's length and
// at steps that start over.
__global__ __launch_bounds__(256) void la_decay_grad(LaArgs a, const float* states,
                                                     const float* adjoints, const float* last_r,
                                                     float* __restrict__ dg, int C) {
  __shared__ double s_e[4];
  __shared__ float s_t[4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, seg = blockIdx.y;
  const int64_t bh = blockIdx.x, ss = (int64_t)a.dk * a.dv;
  const int b = (int)(bh / a.H), h = (int)(bh % a.H);
  const bool final = seg == a.segs - 1;
  const float* S = final ? a.first + bh * ss : states + (bh * (a.segs - 1) + seg) * ss;
  const float* R = final ? (last_r ? last_r + bh * ss : nullptr)
                         : adjoints + (bh * (a.segs - 1) + seg) * ss;
  double E = 0.0;
  if (R) {
    for (int64_t x = tid; x < ss; x += 256) E += (double)S[x] * (double)R[x];
#pragma unroll
    for (int d = 32; d; d /= 2) E += __shfl_xor(E, d);
    if (lane == 0) s_e[w] = E;
    __syncthreads();
    E = (s_e[0] + s_e[1]) + (s_e[2] + s_e[3]);
  }
  int64_t len = a.T;
  if (a.lengths) {
    const int64_t n = a.lengths[b];
    len = n < 0 ? 0 : n < a.T ? n : a.T;
  }
  const int64_t t0 = (int64_t)seg * a.per * C;
  const int64_t t1 = t0 + (int64_t)a.per * C < a.T ? t0 + (int64_t)a.per * C : a.T;
  const float* g = a.g + b * a.gs[0] + h * a.gs[2];
  for (int64_t hi = t1; hi > t0; hi -= 256) {
    const int64_t t = hi - 256 + tid;
    const float e = t >= t0 ? a.e[bh * a.T + t] : 0.f;
    float s = mg_wave_suffix_sum(e);
    if (lane == 0) s_t[w] = s;
    __syncthreads();
    double later = E;
    for (int i = w + 1; i < 4; ++i) later += (double)s_t[i];
    E += ((double)s_t[0] + (double)s_t[1]) + ((double)s_t[2] + (double)s_t[3]);
    if (t >= t0) {
      const bool off = t >= len || (double)g[t * a.gs[1]] * 1.4426950408889634 < -126.0;
      dg[(b * a.T + t) * a.H + h] = off ? 0.f : (float)(later + (double)s);
    }
    __syncthreads();
  }
}

// A key head's gradient: the sum over the heads that share it, in order.
template <typename T>
__global__ __launch_bounds__(256) void la_heads_sum(const float* __restrict__ part,
                                                    T* __restrict__ out, int64_t n, int group,
                                                    int d) {
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (x >= n) return;
  const float* p = part + x / d * group * d + x % d;
  float s = 0.f;
  for (int i = 0; i < group; ++i) s += p[(int64_t)i * d];
  if constexpr (sizeof(T) == 2) out[x] = __builtin_bit_cast(u16, (__bf16)s);
  else out[x] = s;
}

// ---- one token -------------------------------------------------------------------------------
// A workgroup takes 32 columns of a head's state: 8 lanes of 4 columns, 32 groups of rows.
// Bound by the read and write of the state.
struct LaStep {
  const void *q, *k, *v;
  const float *g, *h;
  void* o;
  float* h_out;
  int64_t qs[2], ks[2], vs[2], gs[2];
  int H, group, dk, dv;
  float scale;
};
template <typename T>
__global__ __launch_bounds__(256) void la_step(LaStep a) {
  __shared__ float s_o[32][33];
  const int tid = threadIdx.x, cl = (tid & 7) * 4, rg = tid >> 3;
  const int64_t bh = blockIdx.x;
  const int b = (int)(bh / a.H), h = (int)(bh % a.H), kh = h / a.group;
  const int c = blockIdx.y * 32 + cl, dv = a.dv;
  const T* q = (const T*)a.q + b * a.qs[0] + kh * a.qs[1];
  const T* k = (const T*)a.k + b * a.ks[0] + kh * a.ks[1];
  const T* v = (const T*)a.v + b * a.vs[0] + h * a.vs[1];
  const float decay = expf(a.g[b * a.gs[0] + h * a.gs[1]]);
  const float* S = a.h + bh * (int64_t)a.dk * dv;
  float* So = a.h_out + bh * (int64_t)a.dk * dv;
  float vv[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) vv[i] = c + i < dv ? to_f(v[c + i]) : 0.f;
  const bool wide = dv % 4 == 0 && (((uintptr_t)S | (uintptr_t)So) & 15) == 0;
#pragma unroll 4
  for (int r = rg; r < a.dk; r += 32) {
    const float kr = to_f(k[r]), qr = to_f(q[r]);
    const float* p = S + (int64_t)r * dv + c;
    float* po = So + (int64_t)r * dv + c;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (wide) {
      if (c < dv) {
        const float4 y = *reinterpret_cast<const float4*>(p);
        x[0] = y.x, x[1] = y.y, x[2] = y.z, x[3] = y.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = c + i < dv ? p[i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = decay * x[i] + kr * vv[i];
      o[i] += qr * x[i];
    }
    if (wide) {
      if (c < dv) *reinterpret_cast<float4*>(po) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < dv) po[i] = x[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) s_o[rg][cl + i] = o[i];
  __syncthreads();
  if (tid < 32 && blockIdx.y * 32 + tid < dv) {
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < 32; ++r) s += s_o[r][tid];
    T* out = (T*)a.o + bh * dv + blockIdx.y * 32 + tid;
    if constexpr (sizeof(T) == 2) *out = __builtin_bit_cast(u16, (__bf16)(a.scale * s));
    else *out = a.scale * s;
  }
}

// ---- host ------------------------------------------------------------------------------------
constexpr int LA_MAXD = 128;

bool la_ok(int dtype, int64_t B, int64_t T, int H, int Hk, int dk, int dv) {
  return !(dtype & ~1) && B >= 1 && T >= 1 && H >= 1 && Hk >= 1 && H % Hk == 0 && dk >= 1 &&
         dv >= 1 && dk <= LA_MAXD && dv <= LA_MAXD && H <= (1 << 20) &&
         B * H <= (1ll << 24) && T <= (1ll << 32);
}

struct Plan {
  int C, segs, per;
};
// Segments of a sequence: those that finish first, counting chunks in a row on a CU.  A
// workgroup takes a CU's LDS with heads past 64 wide, half of it otherwise; the pass that
// forms the segments' states costs about half of the main one for each chunk.
Plan la_plan(int dtype, int64_t B, int64_t T, int H, int dk, int dv) {
  const int C = dtype ? 64 : 32;
  const int64_t cap = dk > 64 || dv > 64 ? 256 : 512, BH = B * H, NC = (T + C - 1) / C;
  Plan best = {C, 1, (int)NC};
  double least = 1e300;
  for (int64_t n = 1; n <= 64 && n <= NC; ++n) {
    const int64_t per = (NC + n - 1) / n, segs = (NC + per - 1) / per;
    if (segs != n) continue;
    const double cost = (double)((BH * n + cap - 1) / cap) * per +
                        (n > 1 ? 0.5 * (double)((BH * (n - 1) + cap - 1) / cap) * per + 2.0 : 0.0);
    if (cost < least) least = cost, best = {C, (int)n, (int)per};
  }
  return best;
}

size_t la_bound_bytes(const Plan& p, int64_t BH, int dk, int dv) {
  return mg_align_up((size_t)BH * (p.segs - 1) * dk * dv * sizeof(float), 256);
}
size_t la_decay_bytes(const Plan& p, int64_t BH) {
  return mg_align_up((size_t)BH * (p.segs - 1) * sizeof(float), 256);
}

template <typename T, int C, int DK, int DV>
int la_modes(const LaArgs& a, int mode, int64_t BH, hipStream_t stream) {
  const bool bare = mode == LA_STATE || mode == LA_RSTATE;
  const dim3 grid((unsigned)BH, (unsigned)(a.segs - (bare ? 1 : 0)));
  switch (mode) {
    case LA_STATE: hipLaunchKernelGGL((la_sweep<T, C, DK, DV, LA_STATE>), grid, dim3(NT), 0, stream, a); break;
    case LA_OUT: hipLaunchKernelGGL((la_sweep<T, C, DK, DV, LA_OUT>), grid, dim3(NT), 0, stream, a); break;
    case LA_RSTATE: hipLaunchKernelGGL((la_sweep<T, C, DK, DV, LA_RSTATE>), grid, dim3(NT), 0, stream, a); break;
    case LA_DQ: hipLaunchKernelGGL((la_sweep<T, C, DK, DV, LA_DQ>), grid, dim3(NT), 0, stream, a); break;
    default: hipLaunchKernelGGL((la_sweep<T, C, DK, DV, LA_DKV>), grid, dim3(NT), 0, stream, a);
  }
  return hipGetLastError() == hipSuccess ? MG_OK : MG_ERR_LAUNCH;
}
template <typename T, int C>
int la_sizes(const LaArgs& a, int mode, int64_t BH, hipStream_t stream) {
  if (a.dk <= 64)
    return a.dv <= 64 ? la_modes<T, C, 64, 64>(a, mode, BH, stream)
                      : la_modes<T, C, 64, 128>(a, mode, BH, stream);
  return a.dv <= 64 ? la_modes<T, C, 128, 64>(a, mode, BH, stream)
                    : la_modes<T, C, 128, 128>(a, mode, BH, stream);
}
int la_run(int dtype, const LaArgs& a, int mode, int64_t BH, hipStream_t stream) {
  return dtype ? la_sizes<u16, 64>(a, mode, BH, stream) : la_sizes<float, 32>(a, mode, BH, stream);
}

void la_strides(int64_t (&to)[3], const int64_t* from) {
  for (int i = 0; i < 3; ++i) to[i] = from[i];
}

int la_join_run(const float* first, float* bound, const float* decay, int64_t BH, int64_t ss,
                int n, int rev, hipStream_t stream) {
  hipLaunchKernelGGL(la_join, dim3((unsigned)((BH * ss + 255) / 256)), dim3(256), 0, stream, first,
                     bound, decay, BH, ss, n, rev);
  return hipGetLastError() == hipSuccess ? MG_OK : MG_ERR_LAUNCH;
}

int la_sum_run(int dtype, const float* part, void* out, int64_t n, int group, int d,
               hipStream_t stream) {
  const dim3 grid((unsigned)((n + 255) / 256));
  if (dtype)
    hipLaunchKernelGGL(la_heads_sum<u16>, grid, dim3(256), 0, stream, part, (u16*)out, n, group, d);
  else
    hipLaunchKernelGGL(la_heads_sum<float>, grid, dim3(256), 0, stream, part, (float*)out, n, group,
                       d);
  return hipGetLastError() == hipSuccess ? MG_OK : MG_ERR_LAUNCH;
}

}  // namespace

extern "C" {

size_t mg_linear_attention_state_bytes(int dtype, int64_t B, int64_t T, int H, int Hk, int dk,
                                       int dv) {
  if (!la_ok(dtype, B, T, H, Hk, dk, dv)) return 0;
  const Plan p = la_plan(dtype, B, T, H, dk, dv);
  return 256 + la_bound_bytes(p, B * H, dk, dv) + la_decay_bytes(p, B * H);
}

size_t mg_linear_attention_workspace_bytes(int dtype, int64_t B, int64_t T, int H, int Hk, int dk,
                                           int dv) {
  if (!la_ok(dtype, B, T, H, Hk, dk, dv)) return 0;
  size_t n = mg_linear_attention_state_bytes(dtype, B, T, H, Hk, dk, dv);
  n += mg_align_up((size_t)B * H * T * sizeof(float), 256);
  if (H != Hk) n += (size_t)B * T * H * dk * sizeof(float);
  return n;
}

int mg_linear_attention_fwd(int dtype, const void* q, const void* k, const void* v, const float* g,
                            const int64_t* strides, const int* lengths, const float* h0, void* o,
                            float* hT, void* state, size_t state_bytes, int64_t B, int64_t T,
                            int H, int Hk, int dk, int dv, float scale, hipStream_t stream) {
  if (!q || !k || !v || !g || !strides || !o || !hT || !state ||
      !la_ok(dtype, B, T, H, Hk, dk, dv))
    return MG_ERR_ARG;
  if (state_bytes < mg_linear_attention_state_bytes(dtype, B, T, H, Hk, dk, dv))
    return MG_ERR_WORKSPACE;
  const Plan p = la_plan(dtype, B, T, H, dk, dv);
  const int64_t BH = B * H;
  LaArgs a = {};
  a.q = q, a.k = k, a.v = v, a.g = g, a.lengths = lengths;
  la_strides(a.qs, strides), la_strides(a.ks, strides + 3), la_strides(a.vs, strides + 6);
  la_strides(a.gs, strides + 9);
  a.T = T, a.H = H, a.group = H / Hk, a.dk = dk, a.dv = dv, a.scale = scale;
  a.segs = p.segs, a.per = p.per;
  a.first = h0, a.last = hT, a.out = o;
  a.bound = (float*)state;
  a.decay = (float*)((char*)state + la_bound_bytes(p, BH, dk, dv));
  if (p.segs > 1) {
    int rc = la_run(dtype, a, LA_STATE, BH, stream);
    if (rc == MG_OK)
      rc = la_join_run(h0, a.bound, a.decay, BH, (int64_t)dk * dv, p.segs - 1, 0, stream);
    if (rc != MG_OK) return rc;
  }
  return la_run(dtype, a, LA_OUT, BH, stream);
}

int mg_linear_attention_bwd(int dtype, const void* q, const void* k, const void* v, const float* g,
                            const void* dout, const int64_t* strides, const int* lengths,
                            const float* h0, const float* hT, const void* state, const float* dhT,
                            void* dq, void* dk_, void* dv_, float* dg, float* dh0, int64_t B,
                            int64_t T, int H, int Hk, int dk, int dv, float scale, void* ws,
                            size_t ws_bytes, hipStream_t stream) {
  if (!q || !k || !v || !g || !dout || !strides || !hT || !state || !dq || !dk_ || !dv_ || !dg ||
      !ws || !la_ok(dtype, B, T, H, Hk, dk, dv))
    return MG_ERR_ARG;
  if (ws_bytes < mg_linear_attention_workspace_bytes(dtype, B, T, H, Hk, dk, dv))
    return MG_ERR_WORKSPACE;
  const Plan p = la_plan(dtype, B, T, H, dk, dv);
  const int64_t BH = B * H, ss = (int64_t)dk * dv;
  char* at = (char*)ws;
  LaArgs a = {};
  a.q = q, a.k = k, a.v = v, a.dout = dout, a.g = g, a.lengths = lengths;
  la_strides(a.qs, strides), la_strides(a.ks, strides + 3), la_strides(a.vs, strides + 6);
  la_strides(a.gs, strides + 9), la_strides(a.ds, strides + 12);
  a.T = T, a.H = H, a.group = H / Hk, a.dk = dk, a.dv = dv, a.scale = scale;
  a.segs = p.segs, a.per = p.per;
  float* const adjoints = (float*)at;
  at += la_bound_bytes(p, BH, dk, dv);
  a.decay = (float*)at;
  at += la_decay_bytes(p, BH) + 256;
  a.e = (float*)at;
  at += mg_align_up((size_t)BH * T * sizeof(float), 256);
  float* const part = a.group > 1 ? (float*)at : nullptr;
  // dq, and the queries' side of e, from the first segment on
  a.bound = (float*)state;
  a.first = h0, a.last = nullptr;
  a.out = dq, a.part = part;
  int rc = la_run(dtype, a, LA_DQ, BH, stream);
  if (rc == MG_OK && part) rc = la_sum_run(dtype, part, dq, B * T * Hk * dk, a.group, dk, stream);
  // dk, dv, and the keys' side, from the last one back
  a.bound = adjoints;
  if (rc == MG_OK && p.segs > 1) {
    rc = la_run(dtype, a, LA_RSTATE, BH, stream);
    if (rc == MG_OK) rc = la_join_run(dhT, adjoints, a.decay, BH, ss, p.segs - 1, 1, stream);
  }
  a.first = dhT, a.last = dh0;
  a.out = dk_, a.out2 = dv_;
  if (rc == MG_OK) rc = la_run(dtype, a, LA_DKV, BH, stream);
  if (rc == MG_OK && part) rc = la_sum_run(dtype, part, dk_, B * T * Hk * dk, a.group, dk, stream);
  if (rc != MG_OK) return rc;
  a.first = hT;
  hipLaunchKernelGGL(la_decay_grad, dim3((unsigned)BH, (unsigned)p.segs), dim3(256), 0, stream, a,
                     (const float*)state, (const float*)adjoints, dhT, dg, p.C);
  return hipGetLastError() == hipSuccess ? MG_OK : MG_ERR_LAUNCH;
}

int mg_linear_attention_step(int dtype, const void* q, const void* k, const void* v, const float* g,
                             const int64_t* strides, const float* h, void* o, float* h_out,
                             int64_t B, int H, int Hk, int dk, int dv, float scale,
                             hipStream_t stream) {
  if (!q || !k || !v || !g || !strides || !h || !o || !h_out || (dtype & ~1) || B < 1 || H < 1 ||
      Hk < 1 || H % Hk || dk < 1 || dv < 1 || dk > (1 << 16) || dv > (1 << 16) || H > (1 << 20) ||
      B * H > (1ll << 24))
    return MG_ERR_ARG;
  LaStep a = {};
  a.q = q, a.k = k, a.v = v, a.g = g, a.h = h, a.o = o, a.h_out = h_out;
  for (int i = 0; i < 2; ++i)
    a.qs[i] = strides[i], a.ks[i] = strides[2 + i], a.vs[i] = strides[4 + i], a.gs[i] = strides[6 + i];
  a.H = H, a.group = H / Hk, a.dk = dk, a.dv = dv, a.scale = scale;
  const dim3 grid((unsigned)(B * H), (unsigned)((dv + 31) / 32));
  if (dtype) hipLaunchKernelGGL(la_step<u16>, grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(la_step<float>, grid, dim3(256), 0, stream, a);
  return hipGetLastError() == hipSuccess ? MG_OK : MG_ERR_LAUNCH;
}

}  // extern "C"
