// Softmax cross entropy over a vocabulary, logits never kept (gfx950).
//
//   l_n = W x_n + b,  loss_n = log sum_v exp(l_nv) - l_n[t_n]
//   d_nv = g_n (exp(l_nv - lse_n) - [v = t_n]),  dx = d W,  dW = d^T x,  db = sum_n d_n
//
// Rows whose target is the ignored one are left out at the start: the others are packed one
// after another (their values are never read, so a NaN there stays there), and every launch
// ends at the packed count, which stays on the device.
//
// Forward: one product whose epilogue keeps, for each row and 128 columns of the vocabulary,
// the largest logit and the sum of exponentials against it, and the target's logit; a second
// launch joins them.  Backward, in pieces of the vocabulary: the product again, whose epilogue
// turns the logits into d; then dW's piece and dx's share as products over d, the latter added
// to what the pieces before left, in order, so that memory holds a piece of d and one dx (or a
// few, where the contracted axis is split) however many pieces there are.  So 8 N V D
// operations in place of 6 with kept logits: at D = 1024 a logit's recomputation costs less
// than writing and reading it in fp32.
//
// Products: 256 x 128 tiles of the result, 4 waves of 128 x 64 each with 32 x 32 x 16 matrix
// instructions, 32 contracted elements a step through two LDS buffers (48 KB), so that a CU
// holds two workgroups: one's epilogue, barriers and first loads pass under the other's
// products.  (256 x 256 tiles, one workgroup a CU, spent a third of the logits' products'
// time outside of them.)  Operands are rows of the free index with the contracted one
// consecutive (near), or the other way round (far, read with ds_read_b64_tr_b16): x, W and d
// all lie in memory once, and each is near in one product and far in another.
//
// fp32 inputs are scaled by a power of two that takes the largest finite one (of each row of x, of
// all of W) to 2^14 .. 2^15, and split into two fp16 planes, hi + lo: 22 significant bits down to
// 2^-17 of the largest, then fewer, to 2^-39 of it: an error of the logits far below what fp32
// sums leave.  A product takes the three pairs hi hi, hi lo, lo hi: three times the work of bf16,
// against sixteen times for fp32's own matrix instruction and six for three bf16 planes (24 bits
// at any size; 2047 x 10007 x 392 took 575 us with them, 365 with these).  d's rows, without their
// upstream gradients, are brought to 2^14 .. 2^15 by powers of two from the forward's losses: the
// largest entry is 1 - p of the target.  dW's product sums over rows, so it takes x's rows times
// their upstream gradients over these powers, split again with one scale: what a row adds is held
// to 2^-39 of the largest that a row of the call adds.
// bf16 inputs: d, without the factor of a mean, is rounded to bf16 once; sums are fp32.
// Up to 128 fp32 rows take vocab_few.h's kernels.
// With a bias, x has a column of ones behind its own, which makes db one more column of dW.
#include "mg_common.h"

namespace {

typedef uint16_t u16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int TM = 256, TN = 128, BK = 32, NT = 256;
constexpr int PADK = 64;  // packed rows are padded to this, and the contracted axis to it

// ---- elements --------------------------------------------------------------------------
__device__ __forceinline__ float to_f(u16 x) { return __uint_as_float((unsigned)x << 16); }
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ u16 to_bf(float x) { return __builtin_bit_cast(u16, (__bf16)x); }
__device__ __forceinline__ unsigned pack2(float x, float y) {
  const bf16x2 h = {(__bf16)x, (__bf16)y};
  unsigned u = __builtin_bit_cast(unsigned, h);
  asm("" : "+v"(u));
  return u;
}
// fp16 planes.  What hi leaves for lo; an infinity or NaN is hi's alone.
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ unsigned pack2h(float x, float y) {
  const f16x2 h = {(_Float16)x, (_Float16)y};
  return __builtin_bit_cast(unsigned, h);
}
__device__ __forceinline__ float rest(float x, unsigned pair, int i) {
  const float r = x - (float)__builtin_bit_cast(f16x2, pair)[i];
  return r == r ? r : 0.f;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int d = 32; d; d /= 2) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}
// The power of two that takes `top` to 2^14 .. 2^15, from 2^least to 2^50 (two of them, and a bias
// times both, stay finite); 1 for 0.  Rows of x go down to 2^-100, all of W to 2^-60.
__device__ __forceinline__ float scale_of(float top, int least) {
  if (!(top > 0.f)) return 1.f;
  int e;
  frexpf(top, &e);  // top = m 2^e, m in 1/2 .. 1
  e = 15 - e;
  return ldexpf(1.f, e < least ? least : e > 50 ? 50 : e);
}
constexpr int MAX_PARTS = 256;
// A launch has fewer than 2^32 threads, so a kernel that takes a thread, wave or workgroup for each
// of what a call has many of takes its first workgroup's place among all as well, and more launches
// follow where one is not enough.
constexpr int64_t MAX_THREADS = 1ll << 31;
template <typename F>
void vl_launches(int64_t blocks, int threads, F&& launch) {
  const int64_t most = MAX_THREADS / threads;
  for (int64_t first = 0; first < blocks; first += most)
    launch(dim3((unsigned)(blocks - first < most ? blocks - first : most)), dim3(threads), first);
}
constexpr float ONE_SCALE = 16384.f, D_SCALE = 32768.f;
constexpr int D_LEAST = -16;  // exponent of d's largest entry, below which its own rounding error counts

// ---- packing ----------------------------------------------------------------------------
// Counted rows in order: idx[j] the j-th one's row, pos[i] a row's place or -1, tgt[j] its
// target, -1 where that lies outside the vocabulary; and the left-out rows' losses, 0, if those
// are wanted.  One workgroup.
__global__ __launch_bounds__(1024) void vl_index(const int64_t* __restrict__ target,
                                                 int64_t ignore, int64_t V, int* __restrict__ idx,
                                                 int* __restrict__ pos, int* __restrict__ tgt,
                                                 int* __restrict__ count, float* __restrict__ loss,
                                                 int N) {
  __shared__ int s_n[2][16];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int base = 0, turn = 0;
  // Four rows in a row a thread; the next ones are loaded before the waves meet.
  int64_t t[4], u[4];
  const auto load = [&](int i0, int64_t (&to)[4]) {
#pragma unroll
    for (int x = 0; x < 4; ++x) to[x] = i0 + tid * 4 + x < N ? target[i0 + tid * 4 + x] : ignore;
  };
  load(0, t);
  for (int i0 = 0; i0 < N; i0 += 4096, turn ^= 1) {
    load(i0 + 4096, u);
    int mine = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) mine += t[x] != ignore;
    int sum = mine;  // over the lanes up to this one
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int v = __shfl_up(sum, d);
      if (lane >= d) sum += v;
    }
    if (lane == 63) s_n[turn][w] = sum;
    __syncthreads();
    int at = base + sum - mine;
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      at += x < w ? s_n[turn][x] : 0;
      base += s_n[turn][x];
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = i0 + tid * 4 + x;
      const bool in = t[x] != ignore;
      if (in) idx[at] = i, tgt[at] = t[x] >= 0 && t[x] < V ? (int)t[x] : -1;
      if (i < N) pos[i] = in ? at : -1;
      if (i < N && !in && loss) loss[i] = 0.f;
      at += in;
      t[x] = u[x];
    }
  }
  if (tid == 0) *count = base;
}

// The largest finite magnitude of the (counted) rows, in MAX_PARTS parts.
__global__ __launch_bounds__(1024) void vl_absmax(const float* __restrict__ src, int64_t ld,
                                                 int64_t cols, const int* __restrict__ idx,
                                                 const int* __restrict__ count, int64_t rows,
                                                 float* __restrict__ part) {
  __shared__ float s[16];
  const int64_t n = count ? *count : rows;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  float top = 0.f;
  for (int64_t j = blockIdx.x * 16 + w; j < n; j += MAX_PARTS * 16) {
    const int64_t at = (idx ? (int64_t)idx[j] : j) * ld;
#pragma unroll 4
    for (int64_t c = lane; c < cols; c += 64) {
      const float x = fabsf(src[at + c]);
      top = x < INFINITY ? fmaxf(top, x) : top;
    }
  }
  top = wave_max(top);
  if (lane == 0) s[w] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
    part[blockIdx.x] = top;
  }
}

// Rows of `cols` elements in PL planes, `ld` elements a row, 0 past the columns except a one at
// `ones`.  idx: the counted rows, padded with rows of 0 to a multiple of the contracted step;
// null: all rows.  Two planes are fp16 of the values times the scale that the parts of the
// largest magnitude give or, without them, times a scale of each row's own (written to `scale`; no
// one there), one is bf16.
template <typename E, int PL>
__global__ __launch_bounds__(256) void vl_pack(const E* __restrict__ src, int64_t lds_, int cols,
                                               u16* __restrict__ dst, int ld, int64_t plane,
                                               const int* __restrict__ idx,
                                               const int* __restrict__ count, int64_t rows,
                                               int64_t out_rows, int ones,
                                               const float* __restrict__ top,
                                               float* __restrict__ scale, int64_t first) {
  float by = 1.f;
  if (PL == 2 && top) {
    __shared__ float s_top[4];
    const float t = wave_max(top[threadIdx.x]);
    if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = t;
    __syncthreads();
    by = scale_of(fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3])), -60);
    if (first + blockIdx.x == 0 && threadIdx.x == 0) *scale = by;
  }
  // A wave a row, four elements a lane.
  typedef E E4 __attribute__((ext_vector_type(4), aligned(sizeof(E))));
  const int64_t j = (first + blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t n = count ? *count : rows;
  if (j >= (n + PADK - 1) / PADK * PADK || j >= out_rows) return;
  const bool live = j < n;
  const E* s = src + (live ? (idx ? (int64_t)idx[j] : j) * lds_ : 0);
  if (PL == 2 && !top && live) {
    float most = 0.f;
    for (int c = (threadIdx.x & 63) * 4; c < cols; c += 256) {
      float x[4] = {0.f, 0.f, 0.f, 0.f};
      if (c + 4 <= cols) {
        const E4 y = *reinterpret_cast<const E4*>(s + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = fabsf(to_f(y[e]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < cols) x[e] = fabsf(to_f(s[c + e]));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) most = x[e] < INFINITY ? fmaxf(most, x[e]) : most;
    }
    by = scale_of(wave_max(most), -100);
    if ((threadIdx.x & 63) == 0) scale[j] = by;
  }
  for (int c = (threadIdx.x & 63) * 4; c < ld; c += 256) {
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (live && c + 4 <= cols) {
      const E4 y = *reinterpret_cast<const E4*>(s + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = to_f(y[e]) * by;
    } else if (live) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (c + e < cols) x[e] = to_f(s[c + e]) * by;
        if (PL == 1 && c + e == ones) x[e] = 1.f;
      }
    }
    u16* const to = dst + j * ld + c;
    if constexpr (PL == 1) {
      *reinterpret_cast<uint2*>(to) = make_uint2(pack2(x[0], x[1]), pack2(x[2], x[3]));
    } else {
      const unsigned a = pack2h(x[0], x[1]), b = pack2h(x[2], x[3]);
      *reinterpret_cast<uint2*>(to) = make_uint2(a, b);
      *reinterpret_cast<uint2*>(to + plane) = make_uint2(pack2h(rest(x[0], a, 0), rest(x[1], a, 1)),
                                                         pack2h(rest(x[2], b, 0), rest(x[3], b, 1)));
    }
  }
}

// ---- products -----------------------------------------------------------------------------
enum { VL_LSE = 0, VL_D = 1, VL_OUT = 2 };

struct VlArgs {
  const u16 *A, *B;        // M's and N's operands
  int64_t pa, pb;          // elements between their planes
  const float *sa, *sb;    // fp16 planes: what they were scaled by; LSE and D: sb of each row
  int lda, ldb;            // elements between rows
  int m_rows, n_rows;      // rows (near) or columns (far) that exist; read places are clamped
  const int* m_count;      // on the device, in their place, if not null
  const int* n_count;
  const int* k_count;      // contracted elements on the device, or K
  int K;                   // a multiple of the step
  int ka;                  // of them that a far A has rows for, beside a near B
  int mt, nt, splits;      // tiles, and parts of the contracted axis
  int first, work;         // of all their products, a launch's
  // LSE and D: M the vocabulary from column v0 on, N the packed rows
  int v0, V;               // piece's first column; vocabulary
  const void* bias;
  const int* tgt;
  float2* part;            // LSE: (2 mt, n_ld) largest logit and sum of exponentials
  float* tlogit;           // LSE: the target's logit
  const float2* soft;      // D: of each row, its largest logit and 1 / its sum of exponentials
  const float* g;          // D: of each row, the upstream gradient
  u16* d;                  // D: (planes, n_ld, ldd)
  int64_t pd;
  int ldd, n_ld;
  // OUT: out[n][m]
  void* out;
  int64_t ldo, po;         // elements between rows, between the splits' results
  int m_out, n_out;        // what of it is written
  void* extra;             // column m_out in a vector of its own
  const float* scale;      // of every element, on the device
  int out_f32;
  int add;                 // fp32: out += the product
  int64_t pe;              // extra: elements between the splits'
};

// Fragment of 32 rows (near) or columns (far) x 16 contracted elements.  LDS: near rows of 32
// elements, 16-byte chunk c of row r at c ^ ((r >> 2) & 3); far rows of W (256 or 128), at
// c ^ ((r & 3) << 2).  Both read all 64 banks evenly.
__device__ __forceinline__ int near_place(int r, int c) { return r * BK + ((c ^ ((r >> 2) & 3)) << 3); }
template <int W>
__device__ __forceinline__ int far_place(int r, int c) { return r * W + ((c ^ ((r & 3) << 2)) << 3); }

template <bool FAR, int W>
__device__ __forceinline__ int frag_base() {
  const int l = threadIdx.x & 63;
  if constexpr (FAR)
    return far_place<W>(8 * (l >> 5) + ((l & 15) >> 2), 2 * ((l >> 4) & 1) + ((l & 3) >> 1)) + 4 * (l & 1);
  else
    return near_place(l & 31, l >> 5);
}
// r0: multiple of 32; k0: 0 or 16.
template <bool FAR, int W>
__device__ __forceinline__ bf16x8 frag(const u16* m, int base, int r0, int k0) {
  if constexpr (FAR) {
    typedef __attribute__((address_space(3))) s16x4* lds_t;
    const u16* p = m + (base ^ r0) + k0 * W;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)p);
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(p + 4 * W));
    const s16x8 x = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return __builtin_bit_cast(bf16x8, x);
  } else {
    return *reinterpret_cast<const bf16x8*>(m + (base ^ k0) + r0 * BK);
  }
}

// One operand's step on its way to LDS: W / 64 vectors of 16 bytes a thread, at element offsets
// from the step's first element that hold for every step.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <bool FAR, int W>
__device__ __forceinline__ void step_places(int (&at)[W / 64], int r0, int rows, int ld) {
#pragma unroll
  for (int i = 0; i < W / 64; ++i) {
    const int v = threadIdx.x + i * NT;
    if constexpr (FAR) {
      const int c = r0 + (v % (W / 8)) * 8;
      at[i] = v / (W / 8) * ld + (c + 8 <= rows ? c : 0);
    } else {
      const int r = r0 + (v >> 2);
      at[i] = ((r < rows ? r : rows - 1) - r0) * ld + (v & 3) * 8;
    }
  }
}
// Vector i of a step.  TAIL: a near operand's columns past the `left` ones from p on are 0 (what
// lies there is the next row's).  CLAMP: a far operand's rows past the `left` ones from p on (none or fewer
// in a step that is padding alone) are the last one again: the other operand is 0 there.
template <bool CLAMP, bool TAIL, int W>
__device__ __forceinline__ u32x4 step_load(const u16* p, const int (&at)[W / 64], int i,
                                           int left, int ld) {
  int o = at[i];
  if constexpr (TAIL) {
    // The thread's column is the same in all of its vectors; column 0 of the row stands in.
    const int c = (threadIdx.x & 3) * 8;
    const bool in = c < left;
    const u32x4 x = *reinterpret_cast<const u32x4*>(p + (in ? o : o - c));
    return in ? x : u32x4{0, 0, 0, 0};
  }
  if constexpr (CLAMP) {
    const int over = (int)(threadIdx.x + i * NT) / (W / 8) - (left - 1);
    o -= (over > 0 ? over : 0) * ld;
  }
  return *reinterpret_cast<const u32x4*>(p + o);
}
template <bool FAR, int W>
__device__ __forceinline__ void step_put(u16* m, u32x4 x, int i) {
  const int v = threadIdx.x + i * NT;
  *reinterpret_cast<u32x4*>(m + (FAR ? far_place<W>(v / (W / 8), v % (W / 8)) : near_place(v >> 2, v & 3))) = x;
}

// Pairs of planes in a product, the smaller ones first: lo hi, hi lo, hi hi.
template <int PL>
__device__ __forceinline__ void pair_of(int i, int& a, int& b) {
  a = PL == 2 && i == 0;
  b = PL == 2 && i == 1;
}
template <int PL>
__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
  if constexpr (PL == 2)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

template <int EPI, bool AFAR, bool BFAR, int PL, bool TAIL, typename E>
__global__ __launch_bounds__(NT, 2) void vl_gemm(VlArgs a) {
  __shared__ __align__(16) u16 lds[2][(TM + TN) * BK];  // the buffers: A, then B
  __shared__ __align__(16) float s_bias[TM];
  const int tid = threadIdx.x, lane = tid & 63, wave = mg_uniform(tid >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  // Tiles in bands of 8 along N, so that neighbours share operands; each XCD takes a run.
  const int tiles = a.mt * a.nt;
  int id = blockIdx.x;
  {
    const int per = (a.work + 7) / 8, x = id & 7, y = id >> 3;
    id = x * per + y;
    if (y >= per || id >= a.work) return;
    id += a.first;
  }
  const int split = id / tiles;
  id -= split * tiles;
  const int band = id / (8 * a.mt), in = id - band * 8 * a.mt;
  const int wide = a.nt - band * 8 < 8 ? a.nt - band * 8 : 8;
  const int nt = band * 8 + in % wide, mt = in / wide;
  const int m0 = mt * TM, n0 = nt * TN;
  const int m_rows = a.m_count ? *a.m_count : a.m_rows, n_rows = a.n_count ? *a.n_count : a.n_rows;
  const int K = a.k_count ? (*a.k_count + PADK - 1) / PADK * PADK : a.K;
  if (m0 >= m_rows || n0 >= n_rows) return;

  constexpr int PAIRS = PL == 2 ? 3 : 1;
  const int ksteps = K / BK;
  const int per = (ksteps + a.splits - 1) / a.splits;
  const int s0 = split * per, s1 = s0 + per < ksteps ? s0 + per : ksteps;
  const int steps = s1 > s0 ? (s1 - s0) * PAIRS : 0;

  constexpr int VA = TM / 64, VB = TN / 64;  // vectors of a thread
  u32x4 xa[VA], xb[VB];
  int oa[VA], ob[VB];
  step_places<AFAR, TM>(oa, m0, m_rows, a.lda);
  step_places<BFAR, TN>(ob, n0, n_rows, a.ldb);
  const u16* const A0 = a.A + (AFAR ? 0 : (int64_t)m0 * a.lda);
  const u16* const B0 = a.B + (BFAR ? 0 : (int64_t)n0 * a.ldb);
  // The step being fetched; past the last one it is that one again, so that the loop has no
  // branches.
  int f_k = s0, f_pair = 0, f_left = steps;
  const u16 *fA = nullptr, *fB = nullptr;
  const auto aim = [&]() {
    int p, q;
    pair_of<PL>(f_pair, p, q);
    fA = A0 + p * a.pa + (AFAR ? (int64_t)f_k * BK * a.lda : (int64_t)f_k * BK);
    fB = B0 + q * a.pb + (BFAR ? (int64_t)f_k * BK * a.ldb : (int64_t)f_k * BK);
  };
  const auto advance = [&]() {
    if (--f_left > 0 && ++f_k == s1) f_k = s0, ++f_pair;
    aim();
  };
  // Half a step: the first or second of each thread's vectors.
  const auto load = [&](int half) {
#pragma unroll
    for (int v = half * VA / 2; v < (half + 1) * VA / 2; ++v)
      xa[v] = step_load<AFAR && !BFAR, TAIL, TM>(fA, oa, v, a.ka - f_k * BK, a.lda);
#pragma unroll
    for (int v = half * VB / 2; v < (half + 1) * VB / 2; ++v)
      xb[v] = step_load<false, false, TN>(fB, ob, v, 0, a.ldb);
  };
  const auto put = [&](int s, int half) {
#pragma unroll
    for (int v = half * VA / 2; v < (half + 1) * VA / 2; ++v) step_put<AFAR, TM>(lds[s & 1], xa[v], v);
#pragma unroll
    for (int v = half * VB / 2; v < (half + 1) * VB / 2; ++v)
      step_put<BFAR, TN>(lds[s & 1] + TM * BK, xb[v], v);
  };
  // A row's bias is where its sum starts; past the vocabulary that is -inf, so that such a
  // column's exponentials are 0.
  f32x16 acc[4][2];
  float by[2] = {1.f, 1.f};  // powers of two: what the lane's two rows' sums are scaled by
  if constexpr (EPI != VL_OUT) {
    const int m = m0 + tid;
    s_bias[tid] = m >= m_rows ? -INFINITY : a.bias ? to_f(((const E*)a.bias)[a.v0 + m]) : 0.f;
    if constexpr (PL == 2) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = n0 + wn * 64 + 32 * j + (lane & 31);
        by[j] = *a.sa * a.sb[n < n_rows ? n : n_rows - 1];
      }
    }
    __syncthreads();
    const float* const bw = s_bias + wm * 128 + 4 * (lane >> 5);
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      const float4 b = *reinterpret_cast<const float4*>(bw + 8 * c);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        acc[c >> 2][j][4 * (c & 3)] = b.x * by[j], acc[c >> 2][j][4 * (c & 3) + 1] = b.y * by[j];
        acc[c >> 2][j][4 * (c & 3) + 2] = b.z * by[j], acc[c >> 2][j][4 * (c & 3) + 3] = b.w * by[j];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  }
  // A step has two parts of 16 contracted elements.  Fragments are read one part ahead of the
  // products that use them; a step's operands go to LDS in halves during the two parts before
  // it is needed, and each half of the step after that is loaded into the registers it leaves.
  // The barrier of a step comes before its last part, whose products cover the first reads of
  // the next step.
  const int ab = frag_base<AFAR, TM>(), bb = frag_base<BFAR, TN>();
  bf16x8 fa[2][4], fb[2][2];
  const auto read = [&](const u16* l, int k0, int to) {
#pragma unroll
    for (int i = 0; i < 4; ++i) fa[to][i] = frag<AFAR, TM>(l, ab, wm * 128 + i * 32, k0);
#pragma unroll
    for (int j = 0; j < 2; ++j) fb[to][j] = frag<BFAR, TN>(l + TM * BK, bb, wn * 64 + j * 32, k0);
  };
  const auto part = [&](const u16* l, int k0, int from, int s, int half) {
    read(l, k0, from ^ 1);
    put(s, half);
    if (half == 0) advance();
    load(half);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        acc[i][j] = mma<PL>(fa[from][i], fb[from][j], acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);
  };
  if (steps > 0) {
    aim();
    load(0), load(1);
    put(0, 0), put(0, 1);
    advance();
    load(0), load(1);
    __syncthreads();
    read(lds[0], 0, 0);
    put(1, 0);
    advance();
    load(0);
    for (int s = 0; s < steps; ++s) {
      part(lds[s & 1], 16, 0, s + 1, 1);
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
      part(lds[(s + 1) & 1], 0, 1, s, 0);
    }
  }
  __syncthreads();

  // Lane: column n = n0 + 64 wn + 32 j + (lane & 31) of the result; rows m = m0 + 128 wm +
  // 32 i + 8 q + 4 (lane >> 5) + x in acc[i][j][4 q + x].
  const int half = lane >> 5, mw = m0 + wm * 128 + 4 * half, nw = n0 + wn * 64 + (lane & 31);
  // exp(l) of logits that are still scaled.
  const float unit[2] = {1.f / by[0], 1.f / by[1]};
  const float log2[2] = {1.4426950408889634f * unit[0], 1.4426950408889634f * unit[1]};
  if constexpr (EPI == VL_LSE) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = nw + 32 * j;
      const int t = a.tgt[n < n_rows ? n : n_rows - 1] - a.v0 - mw;
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < 64; ++c) top = fmaxf(top, acc[c >> 4][j][c & 15]);
      if (__ballot(t >= 0 && t < 128 && n < n_rows)) {
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (t == 8 * (c >> 2) + (c & 3) && n < n_rows)
            a.tlogit[n] = acc[c >> 4][j][c & 15] * unit[j];
      }
      top = fmaxf(top, __shfl_xor(top, 32));
      const float ref = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 64; ++c) sum += __builtin_amdgcn_exp2f((acc[c >> 4][j][c & 15] - ref) * log2[j]);
      sum += __shfl_xor(sum, 32);
      // fmaxf drops a NaN; the sum keeps it.
      if (half == 0 && n < n_rows) a.part[(int64_t)(2 * mt + wm) * a.n_ld + n] = make_float2(top * unit[j], sum);
    }
  }
  if constexpr (EPI == VL_D) {
    // In two rounds of 64 rows and for each plane, (64 rows n, 256 columns m) in LDS with chunk
    // c of row r at c ^ (r & 31), then whole rows out.  Rows up to the next multiple of the
    // packing are written, as 0.
    u16* const stage = &lds[0][0];
    const int rows = (n_rows + PADK - 1) / PADK * PADK;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = nw + 32 * j, r = n < n_rows ? n : n_rows - 1;
      const float2 soft = a.soft[r];
      const float g = n < n_rows ? a.g[r] : 0.f, sg = soft.y * g, top = soft.x * by[j];
      const int t = a.tgt[r] - a.v0 - mw;
#pragma unroll
      for (int c = 0; c < 64; ++c) {
        acc[c >> 4][j][c & 15] = __builtin_amdgcn_exp2f((acc[c >> 4][j][c & 15] - top) * log2[j]) * sg;
      }
      if (__ballot(t >= 0 && t < 128)) {
#pragma unroll
        for (int c = 0; c < 64; ++c) acc[c >> 4][j][c & 15] -= t == 8 * (c >> 2) + (c & 3) ? g : 0.f;
      }
      const int sr = wn * 32 + (lane & 31);
#pragma unroll
      for (int q = 0; q < PL; ++q) {
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          f32x16& v = acc[c >> 2][j];
          const int e = 4 * (c & 3);
          const unsigned u0 = PL == 2 ? pack2h(v[e], v[e + 1]) : pack2(v[e], v[e + 1]);
          const unsigned u1 = PL == 2 ? pack2h(v[e + 2], v[e + 3]) : pack2(v[e + 2], v[e + 3]);
          *reinterpret_cast<uint2*>(stage + sr * TM + (((wm * 16 + c) ^ (sr & 31)) << 3) + 4 * half) =
              make_uint2(u0, u1);
          if (q + 1 < PL) {
            v[e] = rest(v[e], u0, 0), v[e + 1] = rest(v[e + 1], u0, 1);
            v[e + 2] = rest(v[e + 2], u1, 0), v[e + 3] = rest(v[e + 3], u1, 1);
          }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int v = tid + u * NT, r2 = v >> 5, c = v & 31;
          const int n2 = n0 + (r2 >> 5) * 64 + 32 * j + (r2 & 31);
          if (n2 < rows && m0 + c * 8 < a.ldd)
            *reinterpret_cast<u32x4*>(a.d + q * a.pd + (int64_t)n2 * a.ldd + m0 + c * 8) =
                *reinterpret_cast<const u32x4*>(stage + r2 * TM + ((c ^ (r2 & 31)) << 3));
        }
        __syncthreads();
      }
    }
  }
  if constexpr (EPI == VL_OUT) {
    const bool f32 = a.out_f32;
    // Apart from `size`, which brings the sums to theirs: the product of both may be below what fp32 holds.
    const float scale = *a.scale, size = PL == 2 ? 1.f / (*a.sa * *a.sb) : 1.f, unit1 = PL == 2 ? 1.f / (ONE_SCALE * *a.sb) : 1.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = nw + 32 * j;
      if (n >= a.n_out) continue;
      const int64_t row = split * a.po + n * a.ldo;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int m = mw + 32 * i + 8 * q;
          float v[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) v[x] = scale * (size * acc[i][j][4 * q + x]);
          if (m + 4 <= a.m_out && (a.ldo & 3) == 0) {
            if (f32) {
              float4* const to = reinterpret_cast<float4*>((float*)a.out + row + m);
              if (a.add) {
                const float4 y = *to;
                v[0] += y.x, v[1] += y.y, v[2] += y.z, v[3] += y.w;
              }
              *to = make_float4(v[0], v[1], v[2], v[3]);
            } else *reinterpret_cast<uint2*>((u16*)a.out + row + m) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
          } else {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              if (m + x < a.m_out) {
                if (f32) ((float*)a.out)[row + m + x] = a.add ? ((float*)a.out)[row + m + x] + v[x] : v[x];
                else ((u16*)a.out)[row + m + x] = to_bf(v[x]);
              } else if (m + x == a.m_out && a.extra) {
                const float e = scale * (unit1 * acc[i][j][4 * q + x]);
                if (f32) ((float*)a.extra)[split * a.pe + n] = e;
                else ((u16*)a.extra)[n] = to_bf(e);
              }
            }
          }
        }
    }
  }
}

// ---- joins ----------------------------------------------------------------------------------
// Rows' largest logits and sums from their parts, and their losses.  64 rows a workgroup, 16 threads each.
__global__ __launch_bounds__(1024) void vl_join(const float2* __restrict__ part,
                                                const float* __restrict__ tlogit,
                                                const int* __restrict__ tgt,
                                                const int* __restrict__ idx,
                                                const int* __restrict__ count, int parts, int ld,
                                                float2* __restrict__ soft,
                                                float* __restrict__ loss,
                                                float* __restrict__ most, int first) {
  __shared__ float2 s[16][64];
  const int r = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int n = (first + blockIdx.x) * 64 + r, rows = *count;
  if (n - r >= rows) return;
  const float2* p = part + (n < rows ? n : rows - 1);
  float top = -INFINITY, sum = 0.f;
#pragma unroll 4
  for (int i = w; i < parts; i += 16) {
    const float2 v = p[(int64_t)i * ld];
    const float m = fmaxf(top, v.x), ref = m == -INFINITY ? 0.f : m;
    sum = sum * __expf(top - ref) + v.y * __expf(v.x - ref);
    top = m;
  }
  s[w][r] = make_float2(top, sum);
  __syncthreads();
  if (w != 0 || n >= rows) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) {
    const float2 v = s[i][r];
    const float m = fmaxf(top, v.x), ref = m == -INFINITY ? 0.f : m;
    sum = sum * __expf(top - ref) + v.y * __expf(v.x - ref);
    top = m;
  }
  // The largest logit and the sum stay apart: their log sum would round at the logits' size.
  const bool in = tgt[n] >= 0;
  soft[n] = make_float2(in ? top : __builtin_nanf(""), 1.f / sum);
  const float l = in ? (top - tlogit[n]) + logf(sum) : __builtin_nanf("");
  loss[idx[n]] = l;
  if (most) most[n] = -expm1f(-l);  // 1 - p of the target: d's largest entry
}

// The counted rows' losses' sum, over the count if `mean`, in a fixed order.  One workgroup.
__global__ __launch_bounds__(1024) void vl_total(const float* __restrict__ loss,
                                                 const int* __restrict__ pos,
                                                 const int* __restrict__ count, int N, int mean,
                                                 float* __restrict__ out) {
  __shared__ double s[16];
  double a[4] = {0.0, 0.0, 0.0, 0.0};
  // Both loads of all four rows go out before a sum; a left-out row's loss is whatever lies there.
  for (int i = threadIdx.x; i < N; i += 4096) {
    float v[4];
    int p[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int x = i + u * 1024 < N ? i + u * 1024 : i;
      v[u] = loss[x], p[u] = i + u * 1024 < N ? pos[x] : -1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) a[u] += p[u] >= 0 ? (double)v[u] : 0.0;
  }
  double t = (a[0] + a[1]) + (a[2] + a[3]);
#pragma unroll
  for (int d = 32; d; d /= 2) t += __shfl_xor(t, d);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    t = 0.0;
    for (int i = 0; i < 16; ++i) t += s[i];
    *out = (float)(mean ? t / (*count > 0 ? *count : 1) : t);
  }
}
// What d is multiplied by in its epilogue (g), and factors for all of it.  reduction: 0 each row's
// own, 1 mean, 2 sum.  A factor for all is kept out of d: one over the count, rounded to bf16 in
// every row's largest entry (the target's), would put all gradients off by the same 2^-9.
// fp16 planes (most not null, the rows' largest entries of d without its upstream gradient) hold d
// over a power of two of each row's own, times D_SCALE, without upstream gradients: rows whose own
// are small would lose their bits beside large ones.  What d lacks, `back`, multiplies dx's rows
// where they are summed; dW's product takes x's rows times `weight`, the same over the power of two
// w_scale, which brings the largest upstream gradient of the counted rows (top, for reduction 0) to
// 1/2 .. 1 (.. 2 at the type's end).
__global__ __launch_bounds__(256) void vl_upstream(const float* __restrict__ up,
                                                   const int* __restrict__ idx,
                                                   const int* __restrict__ count, int reduction,
                                                   const float* __restrict__ most,
                                                   const float* __restrict__ top,
                                                   float* __restrict__ g, float* __restrict__ back,
                                                   float* __restrict__ weight,
                                                   float* __restrict__ scale,
                                                   float* __restrict__ w_scale,
                                                   float* __restrict__ d_scale) {
  const int j = blockIdx.x * 256 + threadIdx.x, n = *count;
  int e = 0;
  if (top) {
    __shared__ float s[4];
    const float t = wave_max(top[threadIdx.x]);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = t;
    __syncthreads();
    frexpf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), &e);
    if (e > 127) e = 127;
  }
  if (j == 0) {
    *scale = reduction == 0 ? 1.f : reduction == 1 ? up[0] / (float)(n > 0 ? n : 1) : up[0];
    *w_scale = top ? ldexpf(1.f, e) : *scale;
    *d_scale = D_SCALE;
  }
  if (j >= n) return;
  const float own = reduction == 0 ? up[idx[j]] : 1.f;
  if (!most) {
    g[j] = own;
    return;
  }
  int k = D_LEAST;
  if (most[j] > 0.f) {
    frexpf(most[j], &k);
    k = k > 0 ? 0 : k < D_LEAST ? D_LEAST : k;
  }
  g[j] = ldexpf(D_SCALE, -k);
  back[j] = ldexpf(own, k);
  weight[j] = ldexpf(own, k - e);
}

// Packed rows in two planes, scaled by sx, times their weights: the largest finite magnitude in
// MAX_PARTS parts (of the high plane: 2^-11 of it off at most, and a plane holds twice what its
// scale makes of it), then in two planes with a scale of their own.  The column of ones becomes the
// weights, times ONE_SCALE.
__device__ __forceinline__ void vl_halves(uint2 u, float (&x)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = (float)__builtin_bit_cast(f16x2, e < 2 ? u.x : u.y)[e & 1];
}
__global__ __launch_bounds__(1024) void vl_weigh_top(const u16* __restrict__ x, int ld, int cols,
                                                    const float* __restrict__ weight,
                                                    const float* __restrict__ sx,
                                                    const int* __restrict__ count,
                                                    float* __restrict__ part) {
  __shared__ float s[16];
  const int n = *count, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  float top = 0.f;
  for (int j = blockIdx.x * 16 + w; j < n; j += MAX_PARTS * 16) {
    const float by = weight[j] / sx[j];
#pragma unroll 4
    for (int c = lane * 4; c < cols; c += 256) {
      float v[4];
      vl_halves(*reinterpret_cast<const uint2*>(x + (int64_t)j * ld + c), v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = fabsf(v[e] * by);
        top = c + e < cols && y < INFINITY ? fmaxf(top, y) : top;
      }
    }
  }
  top = wave_max(top);
  if (lane == 0) s[w] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
    part[blockIdx.x] = top;
  }
}
__global__ __launch_bounds__(256) void vl_weigh(const u16* __restrict__ x, u16* __restrict__ to,
                                                int ld, int64_t plane, int cols,
                                                const float* __restrict__ weight,
                                                const float* __restrict__ sx,
                                                const int* __restrict__ count,
                                                const float* __restrict__ top,
                                                float* __restrict__ scale, int64_t first) {
  __shared__ float s_top[4];
  const float t = wave_max(top[threadIdx.x]);
  if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = t;
  __syncthreads();
  const float by = scale_of(fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3])), -100);
  if (first + blockIdx.x == 0 && threadIdx.x == 0) *scale = by;
  const int64_t j = (first + blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int n = *count;
  if (j >= (n + PADK - 1) / PADK * PADK) return;
  const float g = j < n ? weight[j] : 0.f, f = j < n ? g / sx[j] : 0.f;
  for (int c = (threadIdx.x & 63) * 4; c < ld; c += 256) {
    const u16* const p = x + j * ld + c;
    float hi[4], lo[4], y[4];
    vl_halves(*reinterpret_cast<const uint2*>(p), hi);
    vl_halves(*reinterpret_cast<const uint2*>(p + plane), lo);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      y[e] = c + e < cols ? (hi[e] + lo[e]) * f * by : c + e == cols ? g * ONE_SCALE : 0.f;
    const unsigned a = pack2h(y[0], y[1]), b = pack2h(y[2], y[3]);
    u16* const q = to + j * ld + c;
    *reinterpret_cast<uint2*>(q) = make_uint2(a, b);
    *reinterpret_cast<uint2*>(q + plane) = make_uint2(pack2h(rest(y[0], a, 0), rest(y[1], a, 1)),
                                                      pack2h(rest(y[2], b, 0), rest(y[3], b, 1)));
  }
}
// out[i][c] = sum of the parts' rows, pos[i] if given (0 where that is negative), times by of the same
// row if given.
template <typename E>
__global__ __launch_bounds__(256) void vl_sum(const float* __restrict__ part, int64_t po,
                                              int parts, const int* __restrict__ pos, int64_t n,
                                              int cols, const float* __restrict__ by,
                                              E* __restrict__ out, int64_t first) {
  const int64_t x = ((first + blockIdx.x) * 256 + threadIdx.x) * 4;
  if (x >= n) return;
  if ((cols & 3) == 0) {
    const int64_t i = x / cols, j = pos ? pos[i] : i;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (j >= 0)
#pragma unroll 8
      for (int p = 0; p < parts; ++p) {
        const float4 v = *reinterpret_cast<const float4*>(part + p * po + j * cols + x % cols);
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
      }
    if (by && j >= 0) s.x *= by[j], s.y *= by[j], s.z *= by[j], s.w *= by[j];
    if constexpr (sizeof(E) == 4) *reinterpret_cast<float4*>(out + x) = s;
    else *reinterpret_cast<uint2*>(out + x) = make_uint2(pack2(s.x, s.y), pack2(s.z, s.w));
    return;
  }
  for (int64_t y = x; y < x + 4 && y < n; ++y) {
    const int64_t i = y / cols, j = pos ? pos[i] : i;
    float s = 0.f;
    if (j >= 0)
      for (int p = 0; p < parts; ++p) s += part[p * po + j * cols + y % cols];
    if (by && j >= 0) s *= by[j];
    if constexpr (sizeof(E) == 4) out[y] = s;
    else out[y] = to_bf(s);
  }
}

#include "vocab_few.h"

// ---- host ------------------------------------------------------------------------------------
constexpr int64_t up_to(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

struct Shape {
  int64_t N, V, D, np, kp, dx;  // padded rows, contracted columns, columns of packed x
  int64_t lw;                    // elements between W's rows, as the products read them
  int planes;
  bool own_w;                    // W is packed too
  int few;                       // blocks of 32 rows (1, 2, 4) on vocab_few.h's kernels, or 0
  int64_t ldd;                   // their d's row
};

// Pieces of the vocabulary: as few as keep d in half a gigabyte.
constexpr int64_t VL_D_BYTES = 512ll << 20;

bool vl_shape(int dtype, int64_t N, int64_t V, int64_t D, Shape* s) {
  if ((dtype & ~1) || N < 1 || V < 1 || D < 1 || N > (1 << 30) || V > (1 << 30) || D > (1 << 20))
    return false;
  s->N = N, s->V = V, s->D = D;
  s->np = up_to(N, PADK), s->kp = up_to(D, PADK), s->dx = up_to(D + 1, PADK);
  s->planes = dtype ? 1 : 2;
  s->own_w = dtype == 0 || D % 8 != 0;
  s->lw = s->own_w ? s->kp : D;
  s->ldd = up_to(V, 128);
  s->few = dtype == 0 && N <= FEW && D >= 4 && FEW * s->ldd * 4 <= VL_D_BYTES
               ? (N <= 32 ? 1 : N <= 64 ? 2 : 4) : 0;
  return true;
}
template <typename E>
void vl_sum_run(const float* part, int64_t po, int parts, const int* pos, int64_t n, int64_t cols,
                const float* by, void* out, hipStream_t stream) {
  vl_launches((n / 4 + 256) / 256, 256, [&](dim3 grid, dim3 nt, int64_t first) {
    hipLaunchKernelGGL(vl_sum<E>, grid, nt, 0, stream, part, po, parts, pos, n, (int)cols, by, (E*)out,
                       first);
  });
}
struct State {
  int *idx, *pos, *tgt, *count;
  float2* soft;
  float *sx, *sw;  // scales of the packed planes: of each row of x, of W
  float* most;     // with them: rows' largest entries of d
  u16 *xc, *wc;
  size_t bytes;
};
State vl_state(const Shape& s, void* base) {
  char* p = (char*)base;
  const auto take = [&](int64_t n) {
    char* at = p;
    p += up_to(n, 256);
    return at;
  };
  State t;
  t.count = (int*)take(4);
  const bool own = s.planes == 2 && !s.few;
  t.sx = own ? (float*)take(s.N * 4) : nullptr, t.most = own ? (float*)take(s.N * 4) : nullptr;
  t.sw = (float*)take(4);
  t.idx = (int*)take(s.N * 4), t.pos = (int*)take(s.N * 4), t.tgt = (int*)take(s.N * 4);
  t.soft = (float2*)take(s.N * 8);
  t.xc = (u16*)take(s.few ? 32 * s.few * s.dx * 4 : s.planes * s.np * s.dx * 2);
  t.wc = s.own_w && !s.few ? (u16*)take(s.planes * s.V * s.kp * 2) : nullptr;
  t.bytes = p - (char*)base;
  return t;
}

// ---- few rows --------------------------------------------------------------------------------
int few_tiles(const Shape& s) { return s.few == 1 ? 1 : 2; }  // blocks of 32 columns a workgroup
int64_t few_parts(const Shape& s) { return (s.V + 32 * few_tiles(s) - 1) / (32 * few_tiles(s)); }
// dx's parts: columns of the vocabulary in each, for about two workgroups a CU.
int64_t few_per(const Shape& s) {
  const int64_t tiles = (s.D + 127) / 128, want = (512 + tiles - 1) / tiles;
  return up_to((s.V + want - 1) / want, 32);
}
FewArgs few_args(const Shape& s, const State& t, const void* w, const void* bias) {
  FewArgs a = {};
  a.x = (const float*)t.xc, a.w = (const float*)w, a.bias = (const float*)bias;
  a.ldx = (int)s.dx, a.D = (int)s.D, a.V = (int)s.V, a.ldd = (int)s.ldd, a.parts = (int)few_parts(s);
  a.idx = t.idx, a.tgt = t.tgt, a.count = t.count;
  return a;
}
template <int EPI>
void few_logits(const Shape& s, const FewArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)few_parts(s));
  if (s.few == 2) hipLaunchKernelGGL((vl_few_logits<EPI, 2, 4, 2>), grid, dim3(256), 0, stream, a);
  else if (s.few == 4) hipLaunchKernelGGL((vl_few_logits<EPI, 4, 4, 2>), grid, dim3(256), 0, stream, a);
  else if (EPI == VL_LSE && s.N <= 16)  // d's 32 rows are all written
    hipLaunchKernelGGL((vl_few_logits<VL_LSE, 1, 2, 1>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((vl_few_logits<EPI, 1, 2, 2>), grid, dim3(256), 0, stream, a);
}
template <int NB>
void few_products(const Shape& s, const State& t, const FewArgs& a, float* dx_part, void* dw, void* db,
                  hipStream_t stream) {
  if (dx_part) {
    const int64_t per = few_per(s);
    hipLaunchKernelGGL(vl_few_dx<NB>, dim3((unsigned)((s.D + 127) / 128), (unsigned)((s.V + per - 1) / per)),
                       dim3(256), 0, stream, a.d, a.ldd, a.w, a.V, a.D, (int)s.N, a.count, (int)per, dx_part);
  }
  if (dw) {
    const int64_t tiles = (s.D + 127) / 128, wgs = (s.V + 127) / 128, split = (1024 + wgs - 1) / wgs;
    hipLaunchKernelGGL(vl_few_dw<NB>, dim3((unsigned)wgs, (unsigned)(split < tiles ? split : tiles)),
                       dim3(256), 0, stream, a.d, a.ldd, a.x, a.ldx, a.V, a.D, a.count, (float*)dw,
                       (float*)db);
  }
}

// Parts of the contracted axis for `tiles` result tiles on 256 CUs of two workgroups: the fewest
// steps (about 0.8 us each) in a row, beside what the parts of `size` elements cost to write and
// to add (16 bytes an element, 4 TB/s, and a load after another in a thread: 0.2 us a part).
int vl_splits(int64_t tiles, int64_t steps, int64_t size) {
  int best = 1;
  double least = 1e300;
  for (int s = 1; s <= 128 && (s == 1 || steps / s >= 16); ++s) {
    const double cost = (double)((tiles * s + 511) / 512) * ((steps + s - 1) / s + 8) +
                        (s - 1) * (0.25 + 5e-6 * (double)size);
    if (cost < least) least = cost, best = s;
  }
  return best;
}

struct Back {
  int64_t vp, pieces;   // columns of a piece
  int dx_splits, dw_splits;
  float *g, *scale, *w_scale, *d_scale, *top, *back, *weight, *sxw, *dx_part, *dw_part, *db_part;
  u16 *d, *xw;  // xw: x's packed rows times their weights
  size_t bytes, dx_bytes;  // dx_part is last, and not needed without dx
};
Back vl_back(const Shape& s, void* base) {
  Back b = {};
  if (s.few) {
    const int64_t d = up_to(32 * s.few * s.ldd * 4, 256), per = few_per(s);
    b.d = (u16*)base, b.dx_part = (float*)((char*)base + d);
    b.dx_bytes = (s.V + per - 1) / per * s.N * s.D * 4;
    b.bytes = d + b.dx_bytes;
    return b;
  }
  const int64_t most = VL_D_BYTES / (s.np * 2 * s.planes);
  b.pieces = (s.V + (most > TM ? most : TM) - 1) / (most > TM ? most : TM);
  b.vp = up_to((s.V + b.pieces - 1) / b.pieces, TM);
  b.pieces = (s.V + b.vp - 1) / b.vp;
  const int64_t steps = s.planes == 1 ? 1 : 3;
  b.dx_splits = vl_splits((s.np + TN - 1) / TN * ((s.D + TM - 1) / TM), b.vp / BK * steps, s.N * s.D);
  b.dw_splits = vl_splits(b.vp / TN * ((s.D + TM - 1) / TM), s.np / BK * steps, b.vp * s.D);
  char* p = (char*)base;
  const auto take = [&](int64_t n) {
    char* at = p;
    p += up_to(n, 256);
    return at;
  };
  b.g = (float*)take(s.N * 4);
  b.scale = (float*)take(4), b.w_scale = (float*)take(4), b.d_scale = (float*)take(4);
  b.top = (float*)take(MAX_PARTS * 4);
  b.d = (u16*)take(s.planes * s.np * b.vp * 2);
  if (s.planes == 2) {
    b.back = (float*)take(s.N * 4), b.weight = (float*)take(s.N * 4), b.sxw = (float*)take(4);
    b.xw = (u16*)take(s.planes * s.np * s.dx * 2);
  }
  b.dw_part = b.dw_splits > 1 ? (float*)take(b.dw_splits * b.vp * s.D * 4) : nullptr;
  b.db_part = b.dw_splits > 1 ? (float*)take(b.dw_splits * b.vp * 4) : nullptr;
  b.dx_bytes = b.dx_splits * s.N * s.D * 4;
  b.dx_part = (float*)take(b.dx_bytes);  // pieces add to it one after another
  b.bytes = p - (char*)base;
  return b;
}

template <int EPI, bool AFAR, bool BFAR>
int vl_run(int dtype, VlArgs& a, hipStream_t stream) {
  const int64_t work = (int64_t)a.mt * a.nt * a.splits;
  if (work > (1ll << 30)) return MG_ERR_TOO_LARGE;
  vl_launches(work, NT, [&](dim3 n, dim3 nt, int64_t first) {
    a.first = (int)first, a.work = (int)n.x;
    const dim3 grid((n.x + 7) / 8 * 8);
    // W is read where it lies if its rows are whole vectors; the zeros behind rows that are not
    // whole steps cost selections, so rows that are do without them.
    if (EPI != VL_OUT && dtype && a.lda % BK) {
      if constexpr (EPI != VL_OUT)
        hipLaunchKernelGGL((vl_gemm<EPI, AFAR, BFAR, 1, true, u16>), grid, nt, 0, stream, a);
    } else if (dtype) {
      hipLaunchKernelGGL((vl_gemm<EPI, AFAR, BFAR, 1, false, u16>), grid, nt, 0, stream, a);
    } else {
      hipLaunchKernelGGL((vl_gemm<EPI, AFAR, BFAR, 2, false, float>), grid, nt, 0, stream, a);
    }
  });
  return hipGetLastError() == hipSuccess ? MG_OK : MG_ERR_LAUNCH;
}

// The logits' product: M the vocabulary's columns v0 .. v0 + cols - 1, N the packed rows.
VlArgs vl_logits(const Shape& s, const State& t, const void* w, const void* bias, int64_t v0,
                 int64_t cols) {
  VlArgs a = {};
  a.A = (s.own_w ? t.wc : (const u16*)w) + v0 * s.lw;
  a.lda = (int)s.lw, a.pa = s.V * s.lw;
  a.B = t.xc, a.ldb = (int)s.dx, a.pb = s.np * s.dx;
  a.sa = t.sw, a.sb = t.sx;
  a.m_rows = (int)cols, a.n_count = t.count;
  a.K = (int)up_to(s.lw, BK), a.ka = (int)s.lw;
  a.mt = (int)((cols + TM - 1) / TM), a.nt = (int)((s.np + TN - 1) / TN), a.splits = 1;
  a.v0 = (int)v0, a.V = (int)s.V, a.bias = bias, a.tgt = t.tgt, a.n_ld = (int)s.np;
  return a;
}

int64_t vl_part_rows(const Shape& s) { return 2 * ((s.V + TM - 1) / TM); }

void vl_pack_run(int dtype, const void* src, int64_t ld, int64_t cols, u16* dst, int64_t dld,
                 int64_t plane, const int* idx, const int* count, int64_t rows,
                 int64_t out_rows, int ones, float* top, float* scale, hipStream_t stream) {
  if (top)
    hipLaunchKernelGGL(vl_absmax, dim3(MAX_PARTS), dim3(1024), 0, stream, (const float*)src, ld, cols,
                       idx, count, rows, top);
  vl_launches((out_rows + 3) / 4, 256, [&](dim3 grid, dim3 nt, int64_t first) {
    if (dtype)
      hipLaunchKernelGGL((vl_pack<u16, 1>), grid, nt, 0, stream, (const u16*)src, ld, (int)cols, dst,
                         (int)dld, plane, idx, count, rows, out_rows, ones, (const float*)nullptr,
                         (float*)nullptr, first);
    else
      hipLaunchKernelGGL((vl_pack<float, 2>), grid, nt, 0, stream, (const float*)src, ld, (int)cols, dst,
                         (int)dld, plane, idx, count, rows, out_rows, ones, top, scale, first);
  });
}

}  // namespace

extern "C" {

size_t mg_vocab_loss_state_bytes(int dtype, int64_t N, int64_t V, int64_t D) {
  Shape s;
  return vl_shape(dtype, N, V, D, &s) ? vl_state(s, nullptr).bytes : 0;
}

size_t mg_vocab_loss_fwd_workspace_bytes(int dtype, int64_t N, int64_t V, int64_t D) {
  Shape s;
  if (!vl_shape(dtype, N, V, D, &s)) return 0;
  if (s.few) return s.N * (few_parts(s) * sizeof(float2) + 2 * sizeof(float));
  return vl_part_rows(s) * s.np * sizeof(float2) + (s.np + s.N + MAX_PARTS) * sizeof(float);
}

size_t mg_vocab_loss_bwd_workspace_bytes(int dtype, int64_t N, int64_t V, int64_t D) {
  Shape s;
  return vl_shape(dtype, N, V, D, &s) ? vl_back(s, nullptr).bytes : 0;
}

size_t mg_vocab_loss_bwd_dx_bytes(int dtype, int64_t N, int64_t V, int64_t D) {
  Shape s;
  return vl_shape(dtype, N, V, D, &s) ? vl_back(s, nullptr).dx_bytes : 0;
}

int mg_vocab_loss_fwd(int dtype, const void* x, int64_t ldx, const void* w, const void* bias,
                      const int64_t* target, int64_t ignore_index, int reduction, float* loss,
                      int64_t N, int64_t V, int64_t D, void* state, size_t state_bytes, void* ws,
                      size_t ws_bytes, hipStream_t stream) {
  Shape s;
  if (!x || !w || !target || !loss || !state || !ws || reduction < 0 || reduction > 2 || ldx < D ||
      !vl_shape(dtype, N, V, D, &s))
    return MG_ERR_ARG;
  const State t = vl_state(s, state);
  if (state_bytes < t.bytes || ws_bytes < mg_vocab_loss_fwd_workspace_bytes(dtype, N, V, D))
    return MG_ERR_WORKSPACE;
  float2* const part = (float2*)ws;
  float* const tlogit = (float*)(part + (s.few ? N * few_parts(s) : vl_part_rows(s) * s.np));
  float* const rows = !reduction ? loss : s.few ? tlogit + N : tlogit + s.np + MAX_PARTS;
  float* const zero = reduction ? nullptr : loss;
  const auto finish = [&]() {
    if (reduction)
      hipLaunchKernelGGL(vl_total, dim3(1), dim3(1024), 0, stream, rows, t.pos, t.count, (int)N,
                         (int)(reduction == 1), loss);
    return hipGetLastError() == hipSuccess ? MG_OK : MG_ERR_LAUNCH;
  };
  if (s.few) {
    hipLaunchKernelGGL(vl_few_index, dim3(32 * s.few), dim3(256), 0, stream, target, ignore_index,
                       (int)V, (int)N, (const float*)x, ldx, (int)D, t.idx, t.pos, t.tgt, t.count,
                       zero, (float*)t.xc, (int)s.dx);
    FewArgs a = few_args(s, t, w, bias);
    a.part = part, a.tlogit = tlogit;
    few_logits<VL_LSE>(s, a, stream);
    hipLaunchKernelGGL(vl_few_join, dim3((unsigned)N), dim3(256), 0, stream, part, a.parts, tlogit,
                       t.tgt, t.idx, t.count, t.soft, rows);
    return finish();
  }
  hipLaunchKernelGGL(vl_index, dim3(1), dim3(1024), 0, stream, target, ignore_index, V, t.idx,
                     t.pos, t.tgt, t.count, zero, (int)N);
  vl_pack_run(dtype, x, ldx, D, t.xc, s.dx, s.np * s.dx, t.idx, t.count, N, s.np, (int)D, nullptr, t.sx,
              stream);
  if (s.own_w)
    vl_pack_run(dtype, w, D, D, t.wc, s.kp, V * s.kp, nullptr, nullptr, V, V, -1,
                dtype ? nullptr : tlogit + s.np, t.sw, stream);
  VlArgs a = vl_logits(s, t, w, bias, 0, V);
  a.part = part, a.tlogit = tlogit;
  const int rc = vl_run<VL_LSE, false, false>(dtype, a, stream);
  if (rc != MG_OK) return rc;
  vl_launches((N + 63) / 64, 1024, [&](dim3 grid, dim3 nt, int64_t first) {
    hipLaunchKernelGGL(vl_join, grid, nt, 0, stream, part, tlogit, t.tgt, t.idx, t.count,
                       (int)vl_part_rows(s), (int)s.np, t.soft, rows, t.most, (int)first);
  });
  return finish();
}

int mg_vocab_loss_bwd(int dtype, const void* w, const void* bias, const float* dloss,
                      int reduction, void* dx, void* dw, void* db, int64_t N, int64_t V, int64_t D,
                      const void* state, void* ws, size_t ws_bytes, hipStream_t stream) {
  Shape s;
  if (!w || !dloss || !state || !ws || reduction < 0 || reduction > 2 || (db && !dw) ||
      !vl_shape(dtype, N, V, D, &s))
    return MG_ERR_ARG;
  const State t = vl_state(s, const_cast<void*>(state));
  const Back b = vl_back(s, ws);
  if (ws_bytes < b.bytes - (dx ? 0 : b.dx_bytes)) return MG_ERR_WORKSPACE;
  if (s.few) {
    FewArgs a = few_args(s, t, w, bias);
    a.soft = t.soft, a.up = dloss, a.reduction = reduction, a.d = (float*)b.d;
    few_logits<VL_D>(s, a, stream);
    (s.few == 1 ? few_products<1> : s.few == 2 ? few_products<2> : few_products<4>)(
        s, t, a, dx ? b.dx_part : nullptr, dw, db, stream);
    if (dx)
      vl_sum_run<float>(b.dx_part, N * D, (int)((V + few_per(s) - 1) / few_per(s)), t.pos, N * D, D,
                        nullptr, dx, stream);
    return hipGetLastError() == hipSuccess ? MG_OK : MG_ERR_LAUNCH;
  }
  const int e = dtype ? 2 : 4;
  float* const top = !dtype && reduction == 0 ? b.top : nullptr;
  if (top)
    hipLaunchKernelGGL(vl_absmax, dim3(MAX_PARTS), dim3(1024), 0, stream, dloss, (int64_t)1,
                       (int64_t)1, t.idx, t.count, N, top);
  hipLaunchKernelGGL(vl_upstream, dim3((unsigned)((N + 255) / 256)), dim3(256), 0, stream, dloss,
                     t.idx, t.count, reduction, t.most, top, b.g, b.back, b.weight, b.scale, b.w_scale,
                     b.d_scale);
  if (!dtype && dw) {
    hipLaunchKernelGGL(vl_weigh_top, dim3(MAX_PARTS), dim3(1024), 0, stream, t.xc, (int)s.dx, (int)D,
                       b.weight, t.sx, t.count, b.top);
    vl_launches(s.np / 4, 256, [&](dim3 grid, dim3 nt, int64_t first) {
      hipLaunchKernelGGL(vl_weigh, grid, nt, 0, stream, t.xc, b.xw, (int)s.dx, s.np * s.dx, (int)D,
                         b.weight, t.sx, t.count, b.top, b.sxw, first);
    });
  }
  for (int64_t v0 = 0; v0 < V; v0 += b.vp) {
    const int64_t cols = V - v0 < b.vp ? V - v0 : b.vp, kc = up_to(cols, PADK);
    VlArgs a = vl_logits(s, t, w, bias, v0, cols);
    a.soft = t.soft, a.g = b.g;
    a.d = b.d, a.pd = s.np * b.vp, a.ldd = (int)kc;
    int rc = vl_run<VL_D, false, false>(dtype, a, stream);
    if (rc == MG_OK && dx) {
      VlArgs c = {};
      c.A = a.A, c.lda = a.lda, c.pa = a.pa, c.m_rows = (int)s.lw;
      c.sa = t.sw, c.sb = b.d_scale;
      c.B = b.d, c.ldb = (int)kc, c.pb = a.pd, c.n_count = t.count;
      c.K = (int)kc, c.ka = (int)cols;
      c.mt = (int)((D + TM - 1) / TM), c.nt = (int)((s.np + TN - 1) / TN), c.splits = b.dx_splits;
      c.out = b.dx_part, c.add = v0 > 0;
      c.ldo = D, c.po = N * D, c.m_out = (int)D, c.n_out = (int)N, c.out_f32 = 1, c.scale = b.scale;
      rc = vl_run<VL_OUT, true, false>(dtype, c, stream);
    }
    if (rc == MG_OK && dw) {
      VlArgs c = {};
      c.A = dtype ? t.xc : b.xw, c.lda = (int)s.dx, c.pa = s.np * s.dx, c.m_rows = (int)s.dx;
      c.sa = b.sxw, c.sb = b.d_scale;
      c.B = b.d, c.ldb = (int)kc, c.pb = a.pd, c.n_rows = (int)kc;
      c.k_count = t.count, c.ka = 1 << 30;
      c.mt = (int)((D + (db ? 1 : 0) + TM - 1) / TM), c.nt = (int)((cols + TN - 1) / TN);
      c.splits = b.dw_splits;
      c.ldo = D, c.m_out = (int)D, c.n_out = (int)cols, c.scale = b.w_scale;
      void* const to = (char*)dw + v0 * D * e;
      void* const to_b = db ? (char*)db + v0 * e : nullptr;
      if (b.dw_splits > 1) {
        c.out = b.dw_part, c.po = cols * D, c.out_f32 = 1;
        c.extra = db ? b.db_part : nullptr, c.pe = cols;
      } else {
        c.out = to, c.out_f32 = dtype ? 0 : 1, c.extra = to_b;
      }
      rc = vl_run<VL_OUT, true, true>(dtype, c, stream);
      if (rc == MG_OK && b.dw_splits > 1) {
        for (int k = 0; k < (db ? 2 : 1); ++k) {
          const int64_t n = k ? cols : cols * D;
          const float* const from = k ? b.db_part : b.dw_part;
          (dtype ? vl_sum_run<u16> : vl_sum_run<float>)(from, n, b.dw_splits, nullptr, n, k ? 1 : D, nullptr,
                                                        k ? to_b : to, stream);
        }
      }
    }
    if (rc != MG_OK) return rc;
  }
  if (dx)
    (dtype ? vl_sum_run<u16> : vl_sum_run<float>)(b.dx_part, N * D, b.dx_splits, t.pos, N * D, D,
                                                  b.back, dx, stream);
  return hipGetLastError() == hipSuccess ? MG_OK : MG_ERR_LAUNCH;
}

}  // extern "C"
