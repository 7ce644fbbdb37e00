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
// which keeps the sums finite.  What comes through the state is left out there, by a product in
// which 0 times a NaN or an infinity, that a caller's old state may hold, is 0.  (Tokens that are not
// finite do reach the others of their chunk, through the products' zeros.)
//
// Gradient of g.  G_i enters o_i with do_i.o_i and every later use of k_j v_j^T with -k_j.dk_j:
//   e_i = sum_{j<i} X_ij - sum_{j>i} X_ji + q_i.dq_i^inter - k_i.dk_i^inter,
//   X_ij = scale D_ij (q_i.k_j)(do_i.v_j),
// the diagonal cancelling exactly, and dg_t = sum_{i>=t} e_i + <R_end, S_end> over a segment,
// so that what cancels in the sum is never longer than a segment.  Past the next step that starts
// over all of it cancels but for rounding, so there the sum ends, without <R_end, S_end>: a
// document's gradient holds nothing of the ones behind it.
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
// exact.  Operands that are not inputs are split into bf16 planes, with a product for each.  What
// only feeds bf16 outputs (the C x C matrices, the state in o and dv) into two, 16 significant
// bits, so that the outputs' own rounding is the only one that counts: with one plane they were
// 2.35e-3 off in place of 1.66e-3, prompts of 65536 tokens took 250 us in place of 268 and the
// training pass below 450 in place of 470.  What feeds fp32 outputs (decayed keys and queries into
// the states, the states into the gradient of g) into three, 24 bits: with two the states were
// 2.4e-6 off and the gradient of g 7e-6.
//
// Bound: a wave's own chain of a chunk -- barriers, LDS reads of operand fragments and the vector
// instructions that decay and split them -- with one workgroup a CU past heads 64 wide; memory
// would be a quarter of it.  16 x 2048 tokens of 8 heads of 128, bf16, with gradients: 470 us
// (under a profiler: states 36, o 97, adjoint states 36, dq 143, dk and dv 164; joins 10 each, dg 15).
// One sequence of 65536 tokens, forward: 268 us.  One token of 256 sequences of 16 heads: 112 us,
// 4.8 TB/s of states read and written.
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
  float* e;             // (BH, T): what the queries (keys) add to the gradient of G
};

// ---- elements --------------------------------------------------------------------------
__device__ __forceinline__ float to_f(u16 x) { return __uint_as_float((unsigned)x << 16); }
__device__ __forceinline__ float to_f(float x) { return x; }
// Two values rounded to bf16 by one packed conversion; the empty asm keeps it one.
__device__ __forceinline__ unsigned pack2(float x, float y) {
  const bf16x2 h = {(__bf16)x, (__bf16)y};
  unsigned u = __builtin_bit_cast(unsigned, h);
  asm("" : "+v"(u));
  return u;
}
__device__ __forceinline__ float low(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float high(unsigned u) { return __uint_as_float(u & 0xffff0000u); }

// ---- operands ------------------------------------------------------------------------
// A matrix in LDS has rows of D elements without padding; the 16-byte chunk c of row r lies
// at chunk c ^ swz(r).  swz spreads both kinds of fragment reads over all 64 banks: 16 bytes of
// 16 rows (near), which the LDS serves 16 lanes at a time -- 0-3, 12-15, 20-23 and 24-27
// together, then 4-11, 16-19 and 28-31, then the same of the upper half --, and 16 columns of 4
// rows in turn (far), 32 lanes at a time.
template <typename T>
struct Op;

template <typename T, int D>
__device__ __forceinline__ int place(int r, int c) {
  constexpr int CE = Op<T>::VE;
  return r * D + (((c / CE) ^ Op<T>::template swz<D / CE>(r)) * CE | c % CE);
}

template <>
struct Op<u16> {
  typedef bf16x8 Frag;
  static constexpr int KB = 32, VE = 8, PLANES = 3, HALVES = 2;
  template <int CHUNKS>
  static __device__ __forceinline__ int swz(int r) {
    const int x = ((r >> 2) ^ (r >> 3)) & 1;
    if constexpr (CHUNKS >= 16) return ((r & 3) << 1) | ((r >> 3) & 1) | (x << 3);
    else return (r & 2) | (x << 2) | ((r >> 2) & 1);
  }
  // swz(r) ^ swz(r + 4) of a row r whose bit 2 is clear, in elements.
  template <int D>
  static constexpr int FOUR = (D / VE >= 16 ? 8 : 5) * VE;
  // Lane offsets of fragment reads; row and column of the tile and k0 are added by frag_*.
  template <int D>
  static __device__ __forceinline__ int near_base() {
    const int l = threadIdx.x & 63;
    return place<u16, D>(l & 15, 8 * (l >> 4));
  }
  template <int D>
  static __device__ __forceinline__ int far_base() {
    const int l = threadIdx.x & 63;
    return place<u16, D>(8 * (l >> 4) + ((l & 15) >> 2), 4 * (l & 3));
  }
  // Rows of the free index, the contracted one consecutive.
  template <int D>
  static __device__ __forceinline__ Frag near(const u16* m, int base, int r0, int k0) {
    return *reinterpret_cast<const bf16x8*>(m + (base ^ k0) + r0 * D);
  }
  // Rows of the contracted index: 16 lanes fetch 4 rows x 16 columns and get a column each.
  template <int D>
  static __device__ __forceinline__ Frag far(const u16* m, int base, int c0, int k0) {
    typedef __attribute__((address_space(3))) s16x4* lds_t;
    const u16* p = m + (base ^ c0) + k0 * D;
    const u16* p4 = m + (base ^ c0 ^ FOUR<D>) + (k0 + 4) * D;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)p);
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)p4);
    const s16x8 x = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return __builtin_bit_cast(bf16x8, x);
  }
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  // A fragment times w[contracted index], in planes.
  static __device__ __forceinline__ void scaled(Frag b, const float* w, Frag (&to)[PLANES]) {
    const uint4 u = __builtin_bit_cast(uint4, b);
    const unsigned v[4] = {u.x, u.y, u.z, u.w};
    unsigned o[PLANES][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = low(v[i]) * w[2 * i], y = high(v[i]) * w[2 * i + 1];
#pragma unroll
      for (int p = 0; p < PLANES; ++p) {
        o[p][i] = pack2(x, y);
        x -= low(o[p][i]), y -= high(o[p][i]);
      }
    }
#pragma unroll
    for (int p = 0; p < PLANES; ++p)
      to[p] = __builtin_bit_cast(Frag, make_uint4(o[p][0], o[p][1], o[p][2], o[p][3]));
  }
};

template <>
struct Op<float> {
  typedef f32x4 Frag;
  static constexpr int KB = 16, VE = 4, PLANES = 1, HALVES = 1;
  template <int CHUNKS>
  static __device__ __forceinline__ int swz(int r) {
    return r & 15 & (CHUNKS - 1);
  }
  template <int D>
  static __device__ __forceinline__ int near_base() {
    const int l = threadIdx.x & 63;
    return place<float, D>(l & 15, 4 * (l >> 4));
  }
  template <int D>
  static __device__ __forceinline__ int far_base() {
    const int l = threadIdx.x & 63;
    return place<float, D>(4 * (l >> 4), l & 15);
  }
  template <int D>
  static __device__ __forceinline__ Frag near(const float* m, int base, int r0, int k0) {
    return *reinterpret_cast<const f32x4*>(m + (base ^ k0) + r0 * D);
  }
  template <int D>
  static __device__ __forceinline__ Frag far(const float* m, int base, int c0, int k0) {
    f32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = m[(base ^ c0 ^ (4 * i)) + (k0 + i) * D];
    return x;
  }
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ void scaled(Frag b, const float* w, Frag (&to)[PLANES]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) to[0][i] = b[i] * w[i];
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

// acc[tm][tn] += A B over K contracted elements.  A (free index M) and B (free index N) are
// each near (rows of K elements) or far (rows of LA or LB elements), and come in planes: A[0]
// to A[AP - 1] times B[0], and A[0] times the other planes of B.
template <typename T, typename Ti, int K, bool AFAR, bool BFAR, int LA, int LB, int AP, int BP>
__device__ __forceinline__ void product(f32x4 (&acc)[Ti::TM][Ti::TN], const T* const (&A)[AP],
                                        const T* const (&B)[BP]) {
  if (!Ti::live()) return;
  typedef Op<T> O;
  const int ab = AFAR ? O::template far_base<LA>() : O::template near_base<LA>();
  const int bb = BFAR ? O::template far_base<LB>() : O::template near_base<LB>();
#pragma unroll
  for (int k0 = 0; k0 < K; k0 += O::KB) {
    typename O::Frag a[AP][Ti::TM], b[BP][Ti::TN];
#pragma unroll
    for (int p = 0; p < AP; ++p)
#pragma unroll
      for (int t = 0; t < Ti::TM; ++t)
        a[p][t] = AFAR ? O::template far<LA>(A[p], ab, Ti::m0(t), k0)
                       : O::template near<LA>(A[p], ab, Ti::m0(t), k0);
#pragma unroll
    for (int p = 0; p < BP; ++p)
#pragma unroll
      for (int t = 0; t < Ti::TN; ++t)
        b[p][t] = BFAR ? O::template far<LB>(B[p], bb, Ti::n0(t), k0)
                       : O::template near<LB>(B[p], bb, Ti::n0(t), k0);
#pragma unroll
    for (int p = 0; p < AP + BP - 1; ++p)
#pragma unroll
      for (int i = 0; i < Ti::TM; ++i)
#pragma unroll
        for (int j = 0; j < Ti::TN; ++j)
          acc[i][j] = O::mma(a[p < AP ? p : 0][i], b[p < AP ? 0 : p - AP + 1][j], acc[i][j]);
  }
}

// acc += V^T (w K): rows of the contracted index both, K's (free index N) times w in all planes.
template <typename T, typename Ti, int C, int LV, int LK>
__device__ __forceinline__ void take_up(f32x4 (&acc)[Ti::TM][Ti::TN], const T* V, const T* K,
                                        const float* w) {
  typedef Op<T> O;
  constexpr int PL = O::PLANES, KL = O::KB / 4;  // contracted elements of a lane
  const int ab = O::template far_base<LV>(), bb = O::template far_base<LK>();
  const float* const wl = w + KL * ((threadIdx.x & 63) >> 4);
#pragma unroll
  for (int k0 = 0; k0 < C; k0 += O::KB) {
    typename O::Frag a[Ti::TM], b[Ti::TN][PL];
    float x[KL];
#pragma unroll
    for (int i = 0; i < KL; ++i) x[i] = wl[k0 + i];
#pragma unroll
    for (int t = 0; t < Ti::TN; ++t) O::scaled(O::template far<LK>(K, bb, Ti::n0(t), k0), x, b[t]);
#pragma unroll
    for (int t = 0; t < Ti::TM; ++t) a[t] = O::template far<LV>(V, ab, Ti::m0(t), k0);
#pragma unroll
    for (int p = 0; p < PL; ++p)
#pragma unroll
      for (int i = 0; i < Ti::TM; ++i)
#pragma unroll
        for (int j = 0; j < Ti::TN; ++j) acc[i][j] = O::mma(a[i], b[j][p], acc[i][j]);
  }
}

template <typename Ti>
__device__ __forceinline__ void clear(f32x4 (&acc)[Ti::TM][Ti::TN]) {
#pragma unroll
  for (int i = 0; i < Ti::TM; ++i)
#pragma unroll
    for (int j = 0; j < Ti::TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// Four consecutive elements to LDS, rounded; in planes of 8 bits each, the third returned:
// what is left after each rounding is exact.
__device__ __forceinline__ void put4(u16* p, f32x4 x) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack2(x[0], x[1]), pack2(x[2], x[3]));
}
__device__ __forceinline__ void put4(float* p, f32x4 x) { *reinterpret_cast<f32x4*>(p) = x; }
__device__ __forceinline__ uint2 put4_split(u16* p0, u16* p1, f32x4 x) {
  uint2 u;
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    u = make_uint2(pack2(x[0], x[1]), pack2(x[2], x[3]));
    if (p == 0) *reinterpret_cast<uint2*>(p0) = u;
    if (p == 1) *reinterpret_cast<uint2*>(p1) = u;
    if (p < 2) x[0] -= low(u.x), x[1] -= high(u.x), x[2] -= low(u.y), x[3] -= high(u.y);
  }
  return u;
}
// In two planes, the second returned.
__device__ __forceinline__ uint2 put4_rest(u16* p0, f32x4 x) {
  const uint2 u = make_uint2(pack2(x[0], x[1]), pack2(x[2], x[3]));
  *reinterpret_cast<uint2*>(p0) = u;
  return make_uint2(pack2(x[0] - low(u.x), x[1] - high(u.x)), pack2(x[2] - low(u.y), x[3] - high(u.y)));
}
__device__ __forceinline__ uint2 put4_rest(float*, f32x4) { return make_uint2(0u, 0u); }
__device__ __forceinline__ f32x4 get4(const u16* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  return f32x4{low(u.x), high(u.x), low(u.y), high(u.y)};
}
__device__ __forceinline__ f32x4 get4(const float* p) { return *reinterpret_cast<const f32x4*>(p); }

// Four consecutive elements from column c of a row of d, to memory.  WIDE: d and the row's
// start are multiples of 4 elements.
template <bool WIDE>
__device__ __forceinline__ void store4(u16* p, int c, int d, f32x4 x) {
  if constexpr (WIDE) {
    if (c < d) *reinterpret_cast<uint2*>(p + c) = make_uint2(pack2(x[0], x[1]), pack2(x[2], x[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < d) p[c + i] = __builtin_bit_cast(u16, (__bf16)x[i]);
  }
}
template <bool WIDE>
__device__ __forceinline__ void store4(float* p, int c, int d, f32x4 x) {
  if constexpr (WIDE) {
    if (c < d) *reinterpret_cast<f32x4*>(p + c) = x;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < d) p[c + i] = x[i];
  }
}

// f x, and 0 where f is 0 whatever x is: v_mul_legacy_f32's own rule, an instruction in place of
// the two of a selection.
__device__ float mul_legacy(float, float) __asm("llvm.amdgcn.fmul.legacy");
__device__ __forceinline__ f32x4 times(float f, f32x4 x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = mul_legacy(f, x[i]);
  return x;
}

// A chunk's (C, D) block on its way from memory to LDS, 16 bytes a vector; 0 outside the
// sequence and the d columns.  WIDE: vectors are aligned and lie inside a row or outside it;
// they are loaded from a place inside the block in any case and cleared when they are used,
// since a load under a condition is waited for where the branches meet.
template <typename T, int C, int D, bool WIDE>
struct Block {
  static constexpr int VE = Op<T>::VE, N = C * D / VE / NT;
  static_assert(C * D % (VE * NT) == 0, "whole vectors for every thread");
  uint4 x[N];

  static __device__ __forceinline__ int row(int n) { return (threadIdx.x + n * NT) / (D / VE); }
  static __device__ __forceinline__ int col(int n) {
    return (threadIdx.x + n * NT) % (D / VE) * VE;
  }
  // src: the chunk's first row; ld: elements between rows.
  __device__ __forceinline__ void load(const T* src, int64_t ld, int rows, int d) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int r = row(n), c = col(n);
      if constexpr (WIDE) {
        const unsigned at = (unsigned)(r < rows ? r : rows - 1) * (unsigned)ld + (c < d ? c : 0);
        x[n] = *reinterpret_cast<const uint4*>(src + at);
      } else {
        T e[VE];
#pragma unroll
        for (int i = 0; i < VE; ++i) e[i] = r < rows && c + i < d ? src[r * ld + c + i] : (T)0;
        __builtin_memcpy(&x[n], e, 16);
      }
    }
  }
  __device__ __forceinline__ void mask(int rows, int d) {
    if (WIDE && (rows < C || d < D)) {
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (row(n) >= rows || col(n) >= d) x[n] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  __device__ __forceinline__ void put(T* m) const {
#pragma unroll
    for (int n = 0; n < N; ++n) *reinterpret_cast<uint4*>(m + place<T, D>(row(n), col(n))) = x[n];
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

template <int CTRL>
__device__ __forceinline__ double dpp0(double x) {
  const int2 u = __builtin_bit_cast(int2, x);
  return __builtin_bit_cast(double,
                            make_int2(__builtin_amdgcn_update_dpp(0, u.x, CTRL, 0xf, 0xf, false),
                                      __builtin_amdgcn_update_dpp(0, u.y, CTRL, 0xf, 0xf, false)));
}
__device__ __forceinline__ double lane_of(double x, int l) {
  const int2 u = __builtin_bit_cast(int2, x);
  return __builtin_bit_cast(
      double, make_int2(__builtin_amdgcn_readlane(u.x, l), __builtin_amdgcn_readlane(u.y, l)));
}

// One wave: lane i forms the chunk's i-th gate from its g (0 past the sequence), and the
// factor that its row is taken up into the state with: exp(G_C - G_i) for keys, scale exp(G_i)
// for queries.  The prefix sums take steps of 1, 2, 4 and 8 lanes in each row of 16, then the
// rows' totals.
template <int C, bool REV>
__device__ __forceinline__ void make_gates(Gate* out, float* w, float g, float scale) {
  const int l = threadIdx.x & 63, row = l >> 4;
  constexpr double LOG2E = 1.4426950408889634;
  double s = (double)g * LOG2E;
  const bool over = s < -126.0;
  const float n = mg_wave_prefix_sum(over ? 1.f : 0.f);
  s = over ? 0.0 : s;
  s += dpp0<0x111>(s);
  s += dpp0<0x112>(s);
  s += dpp0<0x114>(s);
  s += dpp0<0x118>(s);
  const double a = lane_of(s, 15), b = lane_of(s, 31), c = lane_of(s, 47);
  s += (row > 0 ? a : 0.0) + (row > 1 ? b : 0.0) + (row > 2 ? c : 0.0);
  const float hi = (float)s;
  const Gate me = {hi, (float)(s - (double)hi), n, 0.f};
  if constexpr (REV) {
    if (l < C) w[l] = scale * span0(me);
  } else {
    const auto last = [](float x) {
      return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), C - 1));
    };
    const Gate end = {last(me.hi), last(me.lo), last(me.n), 0.f};
    if (l < C) w[l] = span(end, me);
  }
  if (l < C) out[l] = me;
}

// ---- the sweep -------------------------------------------------------------------------------
// LDS, in elements.  The plain sweeps fill the next chunk's place while this one's is used (TWO): the
// state passes have two sets of operands; LA_OUT two of the values alone, since its queries, keys
// and state are read by the time that the chunk matrices are there.  (Two whole sets would leave no
// room for the states' second plane: with one, prompt-long took 270 us.)  The gradients' have one
// set; the state's two leading planes lie in S and S1, and once they are read the third lies in S,
// and the second planes of LA_DKV's matrices in S1.
template <typename T, int C, int DK, int DV, int MODE>
struct Lds {
  static constexpr int HV = Op<T>::HALVES;
  static constexpr bool GRAD = MODE == LA_DQ || MODE == LA_DKV;
  static constexpr bool BARE = MODE == LA_STATE || MODE == LA_RSTATE;
  static constexpr int K = 0;  // keys (LA_RSTATE: queries)
  static constexpr int Q = K + C * DK;
  static constexpr int O = Q + (BARE ? 0 : C * DK);
  static constexpr int V = O + (GRAD ? C * DV : 0);  // values (LA_RSTATE: output gradients)
  static constexpr int SET = V + C * DV;
  static constexpr bool TWO = !GRAD;
  static constexpr int NEXT_K = BARE ? SET : 0, NEXT_V = BARE ? SET : TWO ? SET - V : 0;  // to the other place
  // Chunk matrices and states, in two planes each.
  static constexpr int MATS = BARE ? 0 : MODE == LA_DKV ? 2 : HV, STATES = BARE ? 0 : HV;
  static constexpr int P = BARE ? 2 * SET : SET + (TWO ? C * DV : 0);
  static constexpr int P2 = P + (BARE ? 0 : C * C);  // LA_DKV: the second matrix, else P's second plane
  static constexpr int S = P + MATS * C * C;
  static constexpr int S1 = S + (BARE ? 0 : DK * DV);
  static constexpr int SECOND = MODE == LA_DKV && HV > 1 ? 2 * C * C : 0;
  static constexpr int LAST = SECOND > DK * DV ? SECOND : DK * DV;
  static constexpr int BYTES = (S + (STATES > 0 ? DK * DV : 0) + (STATES > 1 ? LAST : 0)) * (int)sizeof(T);
};

// Waves a SIMD: registers for two workgroups a CU where the LDS has room for two.
constexpr int la_waves(int DK, int DV, bool WIDE) { return WIDE && DK <= 64 && DV <= 64 ? 4 : 2; }

template <typename T, int C, int DK, int DV, int MODE, bool WIDE>
__global__ __launch_bounds__(NT, la_waves(DK, DV, WIDE)) void la_sweep(LaArgs a) {
  typedef Lds<T, C, DK, DV, MODE> L;
  constexpr int PL = Op<T>::PLANES;
  constexpr bool REV = MODE == LA_RSTATE || MODE == LA_DKV, BARE = L::BARE, GRAD = L::GRAD, TWO = L::TWO;
  typedef Tiling<DV / 16, DK / 16, DK >= 128 ? 1 : 2> TS;  // the state, transposed: M = dv, N = dk
  typedef Tiling<C / 16, C / 16, 4> TC;    // chunk matrices
  typedef Tiling<DK / 16, C / 16, 4> TK;   // (dk, token)
  typedef Tiling<DV / 16, C / 16, 4> TV;   // (dv, token)
  __shared__ __align__(16) char raw[L::BYTES];
  __shared__ Gate gates[2][C];
  __shared__ __align__(16) float weights[2][C];
  // Sums over the chunk matrices' rows and columns, and rows' products with dq or dk, by wave.
  __shared__ float s_row[4][C], s_col[4][C], s_dot[4][C];
  T* const lds = reinterpret_cast<T*>(raw);
  T *const sP = lds + L::P, *const sP2 = lds + L::P2, *const sS = lds + L::S, *const sS1 = lds + L::S1;

  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = mg_uniform(tid >> 6);
  const int64_t bh = blockIdx.x;
  const int seg = blockIdx.y;
  const int64_t b = bh / a.H;
  const int h = (int)(bh % a.H), kh = h / a.group;
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

  // The state: lane (lg, lr) of tile (i, j) holds S[n0 + lr][m0 + 4 lg .. + 3].
  f32x4 S[TS::TM][TS::TN];
  clear<TS>(S);
  const int64_t ss = (int64_t)dk * dv;
  const auto each_tile = [&](auto&& f) {
#pragma unroll
    for (int i = 0; i < TS::TM; ++i)
#pragma unroll
      for (int j = 0; j < TS::TN; ++j)
        if (TS::live()) f(i, j, TS::n0(j) + lr, TS::m0(i) + 4 * lg);
  };
  const auto each_state = [&](auto&& f) {
    each_tile([&](int i, int j, int r, int c) { f(S[i][j], r, c); });
  };

  Block<T, C, DK, WIDE> bq, bk;
  Block<T, C, DV, WIDE> bv, bo;
  const auto at = [&](int n) { return t0 + (int64_t)(REV ? chunks - 1 - n : n) * C; };
  const auto rows_at = [&](int64_t t) { return (int)(e1 - t < C ? e1 - t : C); };
  const auto fetch = [&](int64_t t) {
    const int rows = rows_at(t);
    if constexpr (MODE != LA_STATE) bq.load(q + t * a.qs[1], a.qs[1], rows, dk);
    if constexpr (MODE != LA_RSTATE) bk.load(k + t * a.ks[1], a.ks[1], rows, dk);
    if constexpr (MODE != LA_RSTATE) bv.load(v + t * a.vs[1], a.vs[1], rows, dv);
    if constexpr (GRAD || MODE == LA_RSTATE) bo.load(dout + t * a.ds[1], a.ds[1], rows, dv);
  };
  // Wave 0 forms the gates one chunk ahead, from decays loaded two chunks ahead.
  const auto decays = [&](int n) {
    const int64_t t = at(n);
    return lane < rows_at(t) ? g[(t + lane) * a.gs[1]] : 0.f;
  };
  const auto gates_of = [&](int n, float x) {
    make_gates<C, REV>(gates[n & 1], weights[n & 1], x, a.scale);
  };
  float g_next = 0.f;
  if (chunks > 0) {
    fetch(at(0));
    if (wave == 0) {
      const float g0 = decays(0);
      if (chunks > 1) g_next = decays(1);
      gates_of(0, g0);
    }
  }
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
        if constexpr (WIDE) {
          const bool in = r < dk && c < dv;
          const f32x4 y = *reinterpret_cast<const f32x4*>(from + (in ? r * dv + c : 0));
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = in ? y[i] : 0.f;
        } else if (r < dk) {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = c + i < dv ? from[r * dv + c + i] : 0.f;
        }
      });
  }
  // A fetched chunk, and the state in its leading planes, into LDS.
  const auto put_chunk = [&](int n) {
    T *const to_k = lds + L::K + (n & 1) * L::NEXT_K, *const to_v = lds + L::V + (n & 1) * L::NEXT_V;
    const int rows = rows_at(at(n));
    if constexpr (MODE != LA_RSTATE) {
      bk.mask(rows, dk), bv.mask(rows, dv);
      bk.put(to_k), bv.put(to_v);
    }
    if constexpr (MODE != LA_STATE) {
      bq.mask(rows, dk);
      bq.put(MODE == LA_RSTATE ? to_k : lds + L::Q);
    }
    if constexpr (GRAD || MODE == LA_RSTATE) {
      bo.mask(rows, dv);
      bo.put(MODE == LA_RSTATE ? to_v : lds + L::O);
    }
  };
  uint2 third[TS::TM][TS::TN];  // the third plane, until there is room for it
  const auto put_state = [&]() {
    each_tile([&](int i, int j, int r, int c) {
      const int p = place<T, DV>(r, c);
      if constexpr (PL > 1) third[i][j] = put4_split(sS + p, sS1 + p, S[i][j]);
      else put4(sS + p, S[i][j]);
    });
  };
  // The finished chunk's part of the gradient of G, once its sums are there.
  const auto put_e = [&](int n) {
    const int64_t t = at(n);
    if (tid < rows_at(t)) {
      float x = 0.f;
#pragma unroll
      for (int u = 0; u < TK::WM; ++u) x += s_dot[u][tid];
      if constexpr (MODE == LA_DQ) {
#pragma unroll
        for (int u = 0; u < TC::WM; ++u) x += s_row[u][tid];
#pragma unroll
        for (int u = 0; u < TC::WN && u < C / 16; ++u) x -= s_col[u][tid];
      }
      a.e[bh * T_ + t + tid] = x;
    }
  };
  if constexpr (TWO)
    if (chunks > 0) {
      put_chunk(0);
      if constexpr (!BARE) put_state();
      if (chunks > 1) fetch(at(1));
    }
  float fall = 1.f;  // the segment's decay so far

  for (int n = 0; n < chunks; ++n) {
    const int64_t t = at(n);
    const int rows = rows_at(t);
    const Gate* const ga = gates[n & 1];
    __syncthreads();  // the gates (and operands) are there; the last chunk's are read
    if constexpr (!TWO) {
      if constexpr (GRAD)
        if (n > 0) put_e(n - 1);
      put_chunk(n);
      if constexpr (!BARE) put_state();
      __syncthreads();
      if (n + 1 < chunks) fetch(at(n + 1));
    }
    const T *const sK = lds + L::K + (n & 1) * L::NEXT_K, *const sV = lds + L::V + (n & 1) * L::NEXT_V;
    const T *const sQ = lds + L::Q, *const sO = lds + L::O;
    const Gate end = ga[C - 1];
    const float keep = span0(end);
    const auto update = [&](const T* rows_v, const T* rows_k) {
#pragma unroll
      for (int i = 0; i < TS::TM; ++i)
#pragma unroll
        for (int j = 0; j < TS::TN; ++j) S[i][j] = times(keep, S[i][j]);
      take_up<T, TS, C, DV, DK>(S, rows_v, rows_k, weights[n & 1]);
      fall *= keep;
    };
    if (wave == 0 && n + 1 < chunks) {
      gates_of(n + 1, g_next);
      if (n + 2 < chunks) g_next = decays(n + 2);
    }
    f32x4 ack[TK::TM][TK::TN], acv[TV::TM][TV::TN];
    uint2 lo[TC::TM][TC::TN], lo2[TC::TM][TC::TN];  // LA_DKV: the matrices' second planes
    if constexpr (!BARE) {
      // Chunk matrices, M the token that is contracted next, N the other: (j, i) towards the
      // queries' side, (i, j) towards the keys'.
      f32x4 A[TC::TM][TC::TN], B[TC::TM][TC::TN];
      clear<TC>(A);
      clear<TC>(B);
      const T *const pq[1] = {sQ}, *const pk[1] = {sK}, *const pv[1] = {sV}, *const po[1] = {sO};
      const T *const ps[1] = {sS};
      if constexpr (REV) {
        product<T, TC, DK, false, false, DK, DK, 1, 1>(A, pq, pk);
        product<T, TC, DV, false, false, DV, DV, 1, 1>(B, po, pv);
      } else {
        product<T, TC, DK, false, false, DK, DK, 1, 1>(A, pk, pq);
        if constexpr (GRAD) product<T, TC, DV, false, false, DV, DV, 1, 1>(B, pv, po);
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
              const float pb = B[im][jn][x] * d;
              p[x] = MODE == LA_DQ ? pb : A[im][jn][x] * d;
              p2[x] = pb;
              if constexpr (MODE == LA_DQ) {
                const float xs = j < i ? A[im][jn][x] * pb : 0.f;
                row += xs;
                col[im][x] += xs;
              }
            }
            const int at_p = place<T, C>(nn, mm);
            if constexpr (PL == 1) {
              put4(sP + at_p, p);
              if constexpr (MODE == LA_DKV) put4(sP2 + at_p, p2);
            } else if constexpr (MODE == LA_DKV) {
              lo[im][jn] = put4_rest(sP + at_p, p), lo2[im][jn] = put4_rest(sP2 + at_p, p2);
            } else {
              *reinterpret_cast<uint2*>(sP2 + at_p) = put4_rest(sP + at_p, p);
            }
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
      // What comes through the state: o's, dq's or dk's and dv's.
      const T* const two[2] = {sS, sS1};
      if constexpr (MODE != LA_DQ) {
        clear<TV>(acv);
        if constexpr (PL > 1) product<T, TV, DK, true, false, DV, DK, 2, 1>(acv, two, REV ? pk : pq);
        else product<T, TV, DK, true, false, DV, DK, 1, 1>(acv, ps, REV ? pk : pq);
      }
      if constexpr (GRAD) {
        clear<TK>(ack);
        if constexpr (PL > 1) product<T, TK, DV, false, false, DV, DV, 2, 1>(ack, two, REV ? pv : po);
        else product<T, TK, DV, false, false, DV, DV, 1, 1>(ack, ps, REV ? pv : po);
      }
    }
    if constexpr (!GRAD) update(sV, sK);
    if constexpr (!BARE) __syncthreads();  // the chunk matrices are there, the state is read

    // Through the plane p of a chunk matrix, added to what is there.
    const auto sum_v = [&](f32x4 (&in)[TV::TM][TV::TN], const T* far, const T* p) {
      const T *const af[1] = {far}, *const pp[1] = {p};
      product<T, TV, C, true, false, DV, C, 1, 1>(in, af, pp);
    };
    const auto sum_k = [&](f32x4 (&in)[TK::TM][TK::TN], const T* p) {
      const T *const af[1] = {REV ? sQ : sK}, *const pp[1] = {p};
      product<T, TK, C, true, false, DK, C, 1, 1>(in, af, pp);
    };
    const auto scale_v = [&](auto&& factor) {
#pragma unroll
      for (int j = 0; j < TV::TN; ++j) {
        const float f = factor(TV::n0(j) + lr);
#pragma unroll
        for (int m = 0; m < TV::TM; ++m) acv[m][j] = times(f, acv[m][j]);
      }
    };
    const auto out_v = [&](T* to) {
      if (TV::live()) {
        T* const base = to + ((b * T_ + t) * a.H + h) * dv;
#pragma unroll
        for (int j = 0; j < TV::TN; ++j) {
          const int i = TV::n0(j) + lr;
          if (i < rows) {
            T* const p = base + (unsigned)i * (unsigned)(a.H * dv);
#pragma unroll
            for (int m = 0; m < TV::TM; ++m) store4<WIDE>(p, TV::m0(m) + 4 * lg, dv, acv[m][j]);
          }
        }
      }
    };
    if constexpr (MODE == LA_OUT) {
      scale_v([&](int i) { return a.scale * span0(ga[i]); });
      sum_v(acv, sV, sP);
      if constexpr (PL > 1) sum_v(acv, sV, sP2);
      out_v((T*)a.out);
    }
    if constexpr (MODE == LA_DKV) {
      scale_v([&](int i) { return span(end, ga[i]); });
      sum_v(acv, sO, sP);
      if constexpr (PL == 1) out_v((T*)a.out2);
    }
    if constexpr (GRAD) {
      // The planes that had no room before: the state's third one, and dk's and dv's matrices' second
      // ones; dq of the chunk itself.
      if constexpr (PL > 1) {
        each_tile([&](int i, int j, int r, int c) {
          *reinterpret_cast<uint2*>(sS + place<T, DV>(r, c)) = third[i][j];
        });
        if constexpr (MODE == LA_DKV)
          if (TC::live())
#pragma unroll
            for (int jn = 0; jn < TC::TN; ++jn)
#pragma unroll
              for (int im = 0; im < TC::TM; ++im) {
                const int at_p = place<T, C>(TC::n0(jn) + lr, TC::m0(im) + 4 * lg);
                *reinterpret_cast<uint2*>(sS1 + at_p) = lo[im][jn];
                *reinterpret_cast<uint2*>(sS1 + C * C + at_p) = lo2[im][jn];
              }
      }
      f32x4 in[TK::TM][TK::TN];
      if constexpr (MODE == LA_DQ) {
        clear<TK>(in);
        sum_k(in, sP);
        if constexpr (PL > 1) sum_k(in, sP2);
      }
      __syncthreads();  // those planes are there
      if constexpr (PL > 1) {
        if constexpr (MODE == LA_DKV) {
          sum_v(acv, sO, sS1);
          out_v((T*)a.out2);
        }
        const T *const third[1] = {sS}, *const rv[1] = {REV ? sV : sO};
        product<T, TK, DV, false, false, DV, DV, 1, 1>(ack, third, rv);
      }
      if (TK::live()) {
#pragma unroll
        for (int j = 0; j < TK::TN; ++j) {
          const int i = TK::n0(j) + lr;
          const float f = REV ? span(end, ga[i]) : a.scale * span0(ga[i]);
          float dot = 0.f;
#pragma unroll
          for (int m = 0; m < TK::TM; ++m) {
            ack[m][j] = times(f, ack[m][j]);
            const f32x4 x = get4((REV ? sK : sQ) + place<T, DK>(i, TK::m0(m) + 4 * lg));
#pragma unroll
            for (int u = 0; u < 4; ++u) dot += ack[m][j][u] * x[u];
            if constexpr (MODE == LA_DQ) ack[m][j] += in[m][j];
          }
          dot = mg_pair_sum<32>(mg_pair_sum<16>(dot));
          if (lane < 16) s_dot[TK::wm()][i] = dot;
        }
      }
      if constexpr (MODE == LA_DKV) {
        sum_k(ack, sP2);
        if constexpr (PL > 1) sum_k(ack, sS1 + C * C);
      }
      if (TK::live()) {
        const int64_t base = ((b * T_ + t) * a.H + h) * dk;
        float* const part = a.part + base;
        T* const out = (T*)a.out + base;
#pragma unroll
        for (int j = 0; j < TK::TN; ++j) {
          const int i = TK::n0(j) + lr;
          const unsigned row = (unsigned)i * (unsigned)(a.H * dk);
          if (i < rows) {
#pragma unroll
            for (int m = 0; m < TK::TM; ++m) {
              const int c = TK::m0(m) + 4 * lg;
              if (a.part) store4<WIDE>(part + row, c, dk, ack[m][j]);
              else store4<WIDE>(out + row, c, dk, ack[m][j]);
            }
          }
        }
      }
      update(REV ? sO : sV, REV ? sQ : sK);
    }
    if (TWO && n + 1 < chunks) {
      if constexpr (!BARE) put_state();
      put_chunk(n + 1);
      if (n + 2 < chunks) fetch(at(n + 2));
    }
  }
  if constexpr (GRAD)
    if (chunks > 0) {
      __syncthreads();
      put_e(chunks - 1);
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
      if (r < dk) store4<WIDE>(to + r * dv, c, dv, x);
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
      for (int64_t x = z0 + tid; x < t1; x += NT) a.e[bh * T_ + x] = 0.f;
    }
    if constexpr (MODE == LA_DKV) zero((T*)a.out2, dv);
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
  // Eight segments' loads at a time: a store to bound ends what the compiler would load ahead.
  for (int i0 = 0; i0 < n; i0 += 8) {
    float y[8], f[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u < n ? i0 + u : n - 1;
      const int64_t seg = bh * n + (rev ? n - 1 - i : i);
      y[u] = bound[seg * ss + at], f[u] = decay[seg];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (i0 + u >= n) break;
      const int64_t seg = bh * n + (rev ? n - 1 - i0 - u : i0 + u);
      s = f[u] == 0.f ? y[u] : f[u] * s + y[u];  // a start in between: as the sweeps
      bound[seg * ss + at] = s;
    }
  }
}

// e: the queries' side less the keys'.  dg_t = sum of e from t up to the next step that starts over,
// or to its segment's end + <R, S> there; 0 past a sequence's length and at steps that start over.
// A workgroup of 16 waves takes a segment: at fewer the product's loads wait for one another
// (4 waves: 35 us at 128 heads of 2048 tokens, 16: 9).
constexpr int DG_NT = 1024, DG_W = DG_NT / MG_WAVE;
__device__ __forceinline__ void la_decay_grad_of(const LaArgs& a, const float* states,
                                                 const float* adjoints, const float* last_r,
                                                 const float* __restrict__ keys,
                                                 float* __restrict__ dg, int C, int64_t bh) {
  __shared__ double s_e[DG_W];
  __shared__ float s_t[DG_W];
  __shared__ int s_over[DG_W];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, seg = blockIdx.y;
  const int ss = a.dk * a.dv;
  const int64_t b = bh / a.H;
  const int h = (int)(bh % a.H);
  const bool final = seg == a.segs - 1;
  const float* S = final ? a.first + bh * ss : states + (bh * (a.segs - 1) + seg) * ss;
  const float* R = final ? (last_r ? last_r + bh * ss : nullptr)
                         : adjoints + (bh * (a.segs - 1) + seg) * ss;
  double E = 0.0;
  if (R) {
#pragma unroll 4
    for (int x = tid; x < ss; x += DG_NT) E += (double)S[x] * (double)R[x];
#pragma unroll
    for (int d = 32; d; d /= 2) E += __shfl_xor(E, d);
    if (lane == 0) s_e[w] = E;
    __syncthreads();
    E = 0.0;
#pragma unroll
    for (int i = 0; i < DG_W; ++i) E += s_e[i];
  }
  int64_t len = a.T;
  if (a.lengths) {
    const int64_t n = a.lengths[b];
    len = n < 0 ? 0 : n < a.T ? n : a.T;
  }
  const int64_t t0 = (int64_t)seg * a.per * C;
  const int64_t t1 = t0 + (int64_t)a.per * C < a.T ? t0 + (int64_t)a.per * C : a.T;
  const float* g = a.g + b * a.gs[0] + h * a.gs[2];
  for (int64_t hi = t1; hi > t0; hi -= DG_NT) {
    const int64_t t = hi - DG_NT + tid;
    const float e = t >= t0 ? a.e[bh * a.T + t] - keys[bh * a.T + t] : 0.f;
    const float gt = t >= t0 ? g[t * a.gs[1]] : 0.f;
    const bool over = t >= t0 && t < len && (double)gt * 1.4426950408889634 < -126.0;
    const uint64_t starts = __ballot(over), after = lane < 63 ? starts >> (lane + 1) : 0;
    const int end = after ? lane + __ffsll((unsigned long long)after) : 64;  // the next start's lane
    float s = e;  // over the lanes from this one on, up to `end`
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const float y = __shfl_down(s, d);
      if (lane + d < end) s += y;
    }
    // What a wave adds to the ones before it, and whether anything behind it does.
    if (lane == 0) s_t[w] = over ? 0.f : s, s_over[w] = starts != 0;
    __syncthreads();
    double later = 0.0;
#pragma unroll
    for (int i = DG_W - 1; i >= 0; --i) {
      if (i == w && end == 64) later = E;
      E = (double)s_t[i] + (s_over[i] ? 0.0 : E);
    }
    if (t >= t0) dg[(b * a.T + t) * a.H + h] = over || t >= len ? 0.f : (float)(later + (double)s);
    __syncthreads();
  }
}

// Pairs past the grid's are taken in turn: a launch has fewer than 2^32 threads.  (The barrier
// that ends the loop over a segment's tokens, of which each has some, frees the LDS for the next.)
constexpr int64_t DG_GRID = 1 << 21;
__global__ __launch_bounds__(DG_NT) void la_decay_grad(LaArgs a, const float* states,
                                                       const float* adjoints, const float* last_r,
                                                       const float* __restrict__ keys,
                                                       float* __restrict__ dg, int C, int64_t BH) {
  for (int64_t bh = blockIdx.x; bh < BH; bh += gridDim.x)
    la_decay_grad_of(a, states, adjoints, last_r, keys, dg, C, bh);
}

// A key head's gradient: the sum over the heads that share it, in order.
constexpr int64_t SUM_GRID = 1 << 23;  // 2^31 threads of the fewer than 2^32 that a launch can have
template <typename T>
__global__ __launch_bounds__(256) void la_heads_sum(const float* __restrict__ part,
                                                    T* __restrict__ out, int64_t n, int group,
                                                    int d) {
  for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < n; x += SUM_GRID * 256) {
    const float* p = part + x / d * group * d + x % d;
    float s = 0.f;
    for (int i = 0; i < group; ++i) s += p[(int64_t)i * d];
    if constexpr (sizeof(T) == 2) out[x] = __builtin_bit_cast(u16, (__bf16)s);
    else out[x] = s;
  }
}

// ---- one token -------------------------------------------------------------------------------
// A workgroup takes 32 columns of a head's state: 8 lanes of 4 columns, 32 groups of rows.
// Bound by the read and write of the state.  A step that starts over, by the sweeps' rule, takes
// nothing from the old state, and does not multiply it by 0: that would keep a NaN or an infinity.
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
  const float g = a.g[b * a.gs[0] + h * a.gs[1]], decay = expf(g);
  const bool over = (double)g * 1.4426950408889634 < -126.0;
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
      x[i] = (over ? 0.f : decay * x[i]) + kr * vv[i];
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
// Pairs of a sequence and a head, each a workgroup of the sweeps: a launch has fewer than 2^32 threads.
constexpr int64_t LA_PAIRS = (1ll << 32) / NT;

bool la_ok(int dtype, int64_t B, int64_t T, int H, int Hk, int dk, int dv) {
  return !(dtype & ~1) && B >= 1 && T >= 1 && H >= 1 && Hk >= 1 && H % Hk == 0 && dk >= 1 &&
         dv >= 1 && dk <= LA_MAXD && dv <= LA_MAXD && H <= (1 << 16) &&
         B < LA_PAIRS && B * H < LA_PAIRS && T <= (1ll << 32);
}

struct Plan {
  int C, segs, per;
};
// Segments of a sequence: those that finish first, counting chunks in a row on a CU and half a
// chunk for a workgroup's start and end.  A workgroup takes a CU's LDS with heads past 64 wide,
// half of it otherwise, where one that has the CU for itself takes 0.6 of the time.  The pass
// that forms the segments' states costs about half of the main one for each chunk; the join, its
// launch and the states' bytes, four times each.  Against every number of segments for 11
// problems of 4 to 256 pairs and 8 to 1024 chunks, what this takes is 3% slower than the
// best at most (144 pairs of 32 chunks: 8 segments 69 us, 1: 91, 32: 106).
Plan la_plan(int dtype, int64_t B, int64_t T, int H, int dk, int dv) {
  const int C = dtype ? 64 : 32;
  const int64_t cap = dk > 64 || dv > 64 ? 256 : 512, BH = B * H, NC = (T + C - 1) / C;
  Plan best = {C, 1, (int)NC};
  double least = 1e300;
  for (int64_t n = 1; n <= 64 && n <= NC; ++n) {
    const int64_t per = (NC + n - 1) / n, segs = (NC + per - 1) / per;
    if (segs != n) continue;
    const auto rounds = [&](int64_t work) {
      const int64_t rest = work % cap;
      return (double)(work / cap) + (rest == 0 ? 0.0 : cap == 512 && rest <= 256 ? 0.6 : 1.0);
    };
    double cost = rounds(BH * n) * (per + 0.5);
    if (n > 1)
      cost += 0.5 * rounds(BH * (n - 1)) * (per + 0.5) + 1.0 + 3.2e-7 * (double)((n - 1) * BH * dk * dv);
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

template <typename T, int C, int DK, int DV, bool WIDE>
int la_modes(const LaArgs& a, int mode, int64_t BH, hipStream_t stream) {
  const bool bare = mode == LA_STATE || mode == LA_RSTATE;
  const dim3 grid((unsigned)BH, (unsigned)(a.segs - (bare ? 1 : 0)));
  switch (mode) {
    case LA_STATE: hipLaunchKernelGGL((la_sweep<T, C, DK, DV, LA_STATE, WIDE>), grid, dim3(NT), 0, stream, a); break;
    case LA_OUT: hipLaunchKernelGGL((la_sweep<T, C, DK, DV, LA_OUT, WIDE>), grid, dim3(NT), 0, stream, a); break;
    case LA_RSTATE: hipLaunchKernelGGL((la_sweep<T, C, DK, DV, LA_RSTATE, WIDE>), grid, dim3(NT), 0, stream, a); break;
    case LA_DQ: hipLaunchKernelGGL((la_sweep<T, C, DK, DV, LA_DQ, WIDE>), grid, dim3(NT), 0, stream, a); break;
    default: hipLaunchKernelGGL((la_sweep<T, C, DK, DV, LA_DKV, WIDE>), grid, dim3(NT), 0, stream, a);
  }
  return hipGetLastError() == hipSuccess ? MG_OK : MG_ERR_LAUNCH;
}
template <typename T, int C, bool WIDE>
int la_sizes(const LaArgs& a, int mode, int64_t BH, hipStream_t stream) {
  if (a.dk <= 64)
    return a.dv <= 64 ? la_modes<T, C, 64, 64, WIDE>(a, mode, BH, stream)
                      : la_modes<T, C, 64, 128, WIDE>(a, mode, BH, stream);
  return a.dv <= 64 ? la_modes<T, C, 128, 64, WIDE>(a, mode, BH, stream)
                    : la_modes<T, C, 128, 128, WIDE>(a, mode, BH, stream);
}
// Rows made of whole aligned 16-byte vectors, close enough that a chunk's offsets fit 32 bits.
bool la_wide(const void* p, const int64_t (&s)[3], int d, int ve) {
  return !p || ((((uintptr_t)p) & 15) == 0 && d % ve == 0 && s[0] % ve == 0 && s[1] % ve == 0 &&
                s[2] % ve == 0 && s[1] >= 0 && s[1] < (1 << 24));
}
int la_run(int dtype, const LaArgs& a, int mode, int64_t BH, hipStream_t stream) {
  const int ve = dtype ? 8 : 4;
  const auto al = [](const void* p) { return (((uintptr_t)p) & 15) == 0; };
  const bool wide = la_wide(a.q, a.qs, a.dk, ve) && la_wide(a.k, a.ks, a.dk, ve) &&
                    la_wide(a.v, a.vs, a.dv, ve) && la_wide(a.dout, a.ds, a.dv, ve) &&
                    al(a.first) && al(a.last) && al(a.bound) && al(a.out) && al(a.out2) && al(a.part);
  if (dtype)
    return wide ? la_sizes<u16, 64, true>(a, mode, BH, stream)
                : la_sizes<u16, 64, false>(a, mode, BH, stream);
  return wide ? la_sizes<float, 32, true>(a, mode, BH, stream)
              : la_sizes<float, 32, false>(a, mode, BH, stream);
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
  const int64_t blocks = (n + 255) / 256;
  const dim3 grid((unsigned)(blocks < SUM_GRID ? blocks : SUM_GRID));
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
  n += 2 * mg_align_up((size_t)B * H * T * sizeof(float), 256);
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
  float* const queries = (float*)at;
  at += mg_align_up((size_t)BH * T * sizeof(float), 256);
  float* const keys = (float*)at;
  at += mg_align_up((size_t)BH * T * sizeof(float), 256);
  float* const part = a.group > 1 ? (float*)at : nullptr;
  // dq, and the queries' side of e, from the first segment on
  a.bound = (float*)state;
  a.first = h0, a.last = nullptr;
  a.out = dq, a.part = part, a.e = queries;
  int rc = la_run(dtype, a, LA_DQ, BH, stream);
  if (rc == MG_OK && part) rc = la_sum_run(dtype, part, dq, B * T * Hk * dk, a.group, dk, stream);
  // dk, dv, and the keys' side, from the last one back
  a.bound = adjoints;
  if (rc == MG_OK && p.segs > 1) {
    rc = la_run(dtype, a, LA_RSTATE, BH, stream);
    if (rc == MG_OK) rc = la_join_run(dhT, adjoints, a.decay, BH, ss, p.segs - 1, 1, stream);
  }
  a.first = dhT, a.last = dh0;
  a.out = dk_, a.out2 = dv_, a.e = keys;
  if (rc == MG_OK) rc = la_run(dtype, a, LA_DKV, BH, stream);
  if (rc == MG_OK && part) rc = la_sum_run(dtype, part, dk_, B * T * Hk * dk, a.group, dk, stream);
  if (rc != MG_OK) return rc;
  a.first = hT, a.e = queries;
  hipLaunchKernelGGL(la_decay_grad, dim3((unsigned)(BH < DG_GRID ? BH : DG_GRID), (unsigned)p.segs),
                     dim3(DG_NT), 0, stream, a, (const float*)state, (const float*)adjoints, dhT, keys,
                     dg, p.C, BH);
  return hipGetLastError() == hipSuccess ? MG_OK : MG_ERR_LAUNCH;
}

int mg_linear_attention_step(int dtype, const void* q, const void* k, const void* v, const float* g,
                             const int64_t* strides, const float* h, void* o, float* h_out,
                             int64_t B, int H, int Hk, int dk, int dv, float scale,
                             hipStream_t stream) {
  if (!q || !k || !v || !g || !strides || !h || !o || !h_out || (dtype & ~1) || B < 1 || H < 1 ||
      Hk < 1 || H % Hk || dk < 1 || dv < 1 || dk > (1 << 16) || dv > (1 << 16) || H > (1 << 20) ||
      B >= (1ll << 24) || B * H >= (1ll << 24))  // 256 threads a pair: fewer than 2^32
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
