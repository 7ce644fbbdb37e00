// The vocabulary loss of a few fp32 rows (vocab_loss.hip's formulas): 1 to 128 of them, where
// reading W bounds the work.  W is read where it lies, in fp32, and nothing is split into planes:
// packing it costs a pass to find its scale and three times its size beside.  The matrix
// instructions are fp32's own, whose time at 64 rows is what reading W takes.
//
// Four waves a workgroup: NB blocks of 32 rows, times 4 / NB parts of the contracted axis, joined
// through LDS in a fixed order.  dx's and dW's products have W's and x's columns across the lanes
// and take their operands from memory straight to registers: a lane's 16 bytes are four columns
// of four instructions, or four contracted elements, numbered as the lanes hold them.
//
// Kernel times: 8 x 33304 x 1000 forward 41 us (W's 133 MB in 28.5, 4.7 TB/s; on planes 163);
// with gradients, 4 x 50557 x 512 126 us (four times 103 MB at the rate of a copy: 80; on planes
// 250), 64 x 18250 x 768 144, 128 of them 253 (90 at fp32's matrix rate).  On planes 129 rows
// take 268, so 128 is where this ends.
#pragma once

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // at any element

constexpr int FEW = 128;

struct FewArgs {
  const float *x, *w, *bias;  // x: packed rows, zeros up to 32 NB of them and up to ldx
  int ldx, D, V, ldd, parts;
  const int *idx, *tgt, *count;
  float2* part;               // (rows, parts) largest logit and sum of exponentials
  float* tlogit;
  const float2* soft;
  const float* up;            // upstream: each row's, or one
  int reduction;
  float* d;                   // (32 NB, ldd)
};

// Counted rows in order, as vl_index has them, and one of them copied by each workgroup (zeros past
// their count).
__global__ __launch_bounds__(256) void vl_few_index(const int64_t* __restrict__ target,
                                                    int64_t ignore, int V, int N,
                                                    const float* __restrict__ x, int64_t ldx, int D,
                                                    int* __restrict__ idx, int* __restrict__ pos,
                                                    int* __restrict__ tgt, int* __restrict__ count,
                                                    float* __restrict__ loss,
                                                    float* __restrict__ to, int ld) {
  __shared__ int s_n[2], s_row;
  const int tid = threadIdx.x, j = blockIdx.x;
  const int64_t t = tid < N ? target[tid] : ignore;
  const bool in = tid < N && t != ignore;
  const uint64_t bits = __ballot(in);
  if (tid == 0) s_row = -1;
  if (tid < FEW && (tid & 63) == 0) s_n[tid >> 6] = __popcll(bits);
  __syncthreads();
  const int at = __popcll(bits & ((1ull << (tid & 63)) - 1)) + (tid >= 64 ? s_n[0] : 0);
  if (in && at == j) s_row = tid;
  if (j == 0 && tid < N) {
    pos[tid] = in ? at : -1;
    if (!in && loss) loss[tid] = 0.f;
    if (in) idx[at] = tid, tgt[at] = t >= 0 && t < V ? (int)t : -1;
    if (tid == 0) *count = s_n[0] + s_n[1];
  }
  __syncthreads();
  const int row = s_row;
  for (int c = tid; c < ld; c += 256) to[(int64_t)j * ld + c] = row >= 0 && c < D ? x[row * ldx + c] : 0.f;
}

// LSE and D.  A workgroup: 16 MI columns of the vocabulary (the instruction's rows), NB blocks of
// 16 NJ rows.  Both operands have the contracted elements in a row, so a lane's fragments are 16
// bytes of 64 rows' places: read from memory like that, each was an access of its own, and the
// caches gave a quarter of their rate (N = 8: 47 us in place of 28.5).  So steps of 32 KP columns go
// through LDS, from registers that hold the next step's; vector c of row r lies at few_slot.
template <int KP>
__device__ __forceinline__ int few_slot(int r, int c) {
  return r * 8 * KP + (KP == 1 ? c ^ (r & 7) : c ^ (r & 7) ^ ((c & 1) << 3));
}
template <int EPI, int NB, int MI, int NJ>
__global__ __launch_bounds__(256) void vl_few_logits(FewArgs a) {
  constexpr int KP = 4 / NB, W = 32 * KP, RW = 16 * MI, RX = 16 * NJ * NB;
  constexpr int VW = RW * 8 * KP / 256, VX = RX * 8 * KP / 256;  // vectors of a thread
  static_assert((KP - 1) * NB * MI * NJ * 64 <= (RW + RX) * 8 * KP, "the join's room");
  __shared__ f32x4 lds[(RW + RX) * 8 * KP];
  f32x4* const lx = lds + RW * 8 * KP;
  const int tid = threadIdx.x, lane = tid & 63, wave = mg_uniform(tid >> 6);
  const int nb = wave % NB, kp = wave / NB, l = lane & 15, h = lane >> 4;
  const int v0 = blockIdx.x * RW, rows = *a.count, n0 = nb * 16 * NJ;
  const float *pw[VW], *px[VX];
  int sw[VW], sx[VX];
  const int c4 = tid % (8 * KP) * 4;  // the column of a thread's vectors
#pragma unroll
  for (int i = 0; i < VW; ++i) {
    const int r = (tid + 256 * i) / (8 * KP), v = v0 + r;
    pw[i] = a.w + (int64_t)(v < a.V ? v : a.V - 1) * a.D + c4;
    sw[i] = few_slot<KP>(r, c4 / 4);
  }
#pragma unroll
  for (int i = 0; i < VX; ++i) {
    const int r = (tid + 256 * i) / (8 * KP);
    px[i] = a.x + (int64_t)r * a.ldx + c4;
    sx[i] = few_slot<KP>(r, c4 / 4);
  }
  f32x4 acc[MI][NJ], yw[VW], yx[VX];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const auto load = [&](int k) {
#pragma unroll
    for (int i = 0; i < VW; ++i) yw[i] = *reinterpret_cast<const f32x4u*>(pw[i] + k);
#pragma unroll
    for (int i = 0; i < VX; ++i) yx[i] = *reinterpret_cast<const f32x4*>(px[i] + k);
  };
  const auto put = [&]() {
#pragma unroll
    for (int i = 0; i < VW; ++i) lds[sw[i]] = yw[i];
#pragma unroll
    for (int i = 0; i < VX; ++i) lx[sx[i]] = yx[i];
  };
  const auto mul = [&]() {
    if (n0 >= rows) return;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      f32x4 fw[MI], fx[NJ];
#pragma unroll
      for (int i = 0; i < MI; ++i) fw[i] = lds[few_slot<KP>(16 * i + l, 8 * kp + 4 * g + h)];
#pragma unroll
      for (int j = 0; j < NJ; ++j) fx[j] = lx[few_slot<KP>(n0 + 16 * j + l, 8 * kp + 4 * g + h)];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fw[i][e], fx[j][e], acc[i][j], 0, 0, 0);
    }
  };
  const int whole = a.D / W;
  if (whole) load(0);
  for (int c = 0; c < whole; ++c) {
    put();
    __syncthreads();
    load((c + 1 < whole ? c + 1 : c) * W);
    mul();
    __syncthreads();
  }
  if (a.D % W) {  // 0 past the last column
    const int k = whole * W;
#pragma unroll
    for (int i = 0; i < VW; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) yw[i][e] = k + c4 + e < a.D ? pw[i][k + e] : 0.f;
#pragma unroll
    for (int i = 0; i < VX; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) yx[i][e] = k + c4 + e < a.D ? px[i][k + e] : 0.f;
    put();
    __syncthreads();
    mul();
    __syncthreads();
  }
  if constexpr (KP > 1) {
    if (kp > 0) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) lds[(((kp - 1) * NB + nb) * MI * NJ + i * NJ + j) * 64 + lane] = acc[i][j];
    }
    __syncthreads();
    if (kp > 0) return;
#pragma unroll
    for (int p = 1; p < KP; ++p)
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const f32x4 y = lds[(((p - 1) * NB + nb) * MI * NJ + i * NJ + j) * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] += y[e];
        }
  }
  // Row n0 + 16 j + l, columns v0 + 16 i + 4 h + e in acc[i][j][e].  Past the vocabulary -inf.
  const float log2 = 1.4426950408889634f;
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int v = v0 + 16 * i + 4 * h + e;
      const float b = a.bias && v < a.V ? a.bias[v] : 0.f;
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j][e] = v < a.V ? acc[i][j][e] + b : -INFINITY;
    }
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int n = n0 + 16 * j + l, r = n < rows ? n : 0, t = a.tgt[r] - v0 - 4 * h;
    if constexpr (EPI == VL_LSE) {
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          top = fmaxf(top, acc[i][j][e]);
          if (t == 16 * i + e && n < rows) a.tlogit[n] = acc[i][j][e];
        }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float ref = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += __builtin_amdgcn_exp2f((acc[i][j][e] - ref) * log2);
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (h == 0 && n < rows) a.part[(int64_t)n * a.parts + blockIdx.x] = make_float2(top, sum);
    } else {
      const float2 soft = a.soft[r];
      float g = a.reduction ? a.up[0] : rows > 0 ? a.up[a.idx[r]] : 0.f;
      if (a.reduction == 1) g /= (float)(rows > 0 ? rows : 1);
      const float sg = soft.y * g;
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[e] = __builtin_amdgcn_exp2f((acc[i][j][e] - soft.x) * log2) * sg - (t == 16 * i + e ? g : 0.f);
          y[e] = n < rows ? y[e] : 0.f;
        }
        *reinterpret_cast<f32x4*>(a.d + (int64_t)n * a.ldd + v0 + 16 * i + 4 * h) = y;
      }
    }
  }
}

// A row's largest logit and sum from its parts, and its loss.
__global__ __launch_bounds__(256) void vl_few_join(const float2* __restrict__ part, int parts,
                                                   const float* __restrict__ tlogit,
                                                   const int* __restrict__ tgt,
                                                   const int* __restrict__ idx,
                                                   const int* __restrict__ count,
                                                   float2* __restrict__ soft,
                                                   float* __restrict__ loss) {
  __shared__ float2 s[256];
  const int n = blockIdx.x, tid = threadIdx.x;
  if (n >= *count) return;
  const auto join = [](float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x), ref = m == -INFINITY ? 0.f : m;
    return make_float2(m, a.y * __expf(a.x - ref) + b.y * __expf(b.x - ref));
  };
  float2 v = make_float2(-INFINITY, 0.f);
  for (int i = tid; i < parts; i += 256) v = join(v, part[(int64_t)n * parts + i]);
  s[tid] = v;
  __syncthreads();
#pragma unroll
  for (int d = 128; d; d /= 2) {
    if (tid < d) s[tid] = join(s[tid], s[tid + d]);
    __syncthreads();
  }
  if (tid) return;
  v = s[0];
  const bool in = tgt[n] >= 0;
  soft[n] = make_float2(in ? v.x : __builtin_nanf(""), 1.f / v.y);
  loss[idx[n]] = in ? (v.x - tlogit[n]) + logf(v.y) : __builtin_nanf("");
}

// Where a lane's four columns are, of D >= 4: the last ones lie over their neighbours', and both
// lanes compute and write the same.
__device__ __forceinline__ int few_column(int c, int D) { return c + 4 <= D ? c : D - 4; }

// dx's parts: (rows, 128 columns) over `per` columns of the vocabulary (a multiple of 32).
template <int NB>
__global__ __launch_bounds__(256) void vl_few_dx(const float* __restrict__ d, int ldd,
                                                 const float* __restrict__ w, int V, int D, int N,
                                                 const int* __restrict__ count, int per,
                                                 float* __restrict__ part) {
  constexpr int VP = 4 / NB;
  __shared__ float s_acc[VP > 1 ? VP - 1 : 1][NB][4][VP > 1 ? 16 : 1][64];
  const int lane = threadIdx.x & 63, wave = mg_uniform(threadIdx.x >> 6);
  const int nb = wave % NB, vp = wave / NB, l = lane & 31, h = lane >> 5;
  const int rows = *count, col = few_column(blockIdx.x * 128 + 4 * l, D);
  const int first = blockIdx.y * per + vp * (per / VP);
  const int last = (V + 7) / 8 * 8 < first + per / VP ? (V + 7) / 8 * 8 : first + per / VP;
  const float* const dr = d + (int64_t)(nb * 32 + l) * ldd + 4 * h;
  // 8 columns of the vocabulary: v + 4 h + e in vector e of W and element e of d, which is 0 past
  // the last one.
  const auto load = [&](f32x4 (&y)[4], f32x4& g, int v) {
    g = *reinterpret_cast<const f32x4*>(dr + v);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = v + 4 * h + e;
      y[e] = *reinterpret_cast<const f32x4u*>(w + (int64_t)(at < V ? at : V - 1) * D + col);
    }
  };
  f32x16 acc[4];
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[b][e] = 0.f;
  const auto mul = [&](const f32x4 (&y)[4], f32x4 g) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        acc[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(g[e], y[e][b], acc[b], 0, 0, 0);
  };
  if (nb * 32 < rows && first < last) {
    f32x4 y[3][4], g[3];
    const auto clamp = [&](int v) { return v < last ? v : last - 8; };
    load(y[0], g[0], first);
    load(y[1], g[1], clamp(first + 8));
    for (int v = first;;) {
#pragma unroll
      for (int u = 0; u < 3; ++u) {
        load(y[(u + 2) % 3], g[(u + 2) % 3], clamp(v + 16));
        mul(y[u], g[u]);
        v += 8;
        if (v >= last) goto done;
      }
    }
  }
done:
  if constexpr (VP > 1) {
    if (vp > 0) {
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) s_acc[vp - 1][nb][b][e][lane] = acc[b][e];
    }
    __syncthreads();
    if (vp > 0) return;
#pragma unroll
    for (int p = 1; p < VP; ++p)
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[b][e] += s_acc[p - 1][nb][b][e][lane];
  }
  // Rows 8 q + 4 h + x of the block in acc[b][4 q + x], column col + b.
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int n = nb * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
    if (n < N)
      *reinterpret_cast<f32x4u*>(part + ((int64_t)blockIdx.y * N + n) * D + col) =
          f32x4{acc[0][e], acc[1][e], acc[2][e], acc[3][e]};
  }
}

// dW and db: a wave takes 32 columns of the vocabulary and every gridDim.y-th 128 columns of W.
template <int NB>
__global__ __launch_bounds__(256) void vl_few_dw(const float* __restrict__ d, int ldd,
                                                 const float* __restrict__ x, int ldx, int V, int D,
                                                 const int* __restrict__ count,
                                                 float* __restrict__ dw, float* __restrict__ db) {
  const int lane = threadIdx.x & 63, wave = mg_uniform(threadIdx.x >> 6);
  const int l = lane & 31, h = lane >> 5, v0 = (blockIdx.x * 4 + wave) * 32;
  if (v0 >= V) return;
  const int blocks = (*count + 31) / 32;
  float g[NB][16];  // d of rows 32 i + 2 k + h, column v0 + l
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int k = 0; k < 16; ++k) g[i][k] = d[(int64_t)(32 * i + 2 * k + h) * ldd + v0 + l];
  if (db && blockIdx.y == 0) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int k = 0; k < 16; ++k) s += g[i][k];
    s += __shfl_xor(s, 32);
    if (h == 0 && v0 + l < V) db[v0 + l] = s;
  }
  for (int t = blockIdx.y; t * 128 < D; t += gridDim.y) {
    const int col = few_column(t * 128 + 4 * l, D);
    const float* const xr = x + (int64_t)h * ldx + col;
    f32x16 acc[4];
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[b][e] = 0.f;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      if (i < blocks) {
        f32x4 y[16];
#pragma unroll
        for (int k = 0; k < 16; ++k)
          y[k] = *reinterpret_cast<const f32x4u*>(xr + (int64_t)(32 * i + 2 * k) * ldx);
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
          for (int b = 0; b < 4; ++b)
            acc[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(g[i][k], y[k][b], acc[b], 0, 0, 0);
      }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int v = v0 + 8 * (e >> 2) + 4 * h + (e & 3);
      if (v < V)
        *reinterpret_cast<f32x4u*>(dw + (int64_t)v * D + col) = f32x4{acc[0][e], acc[1][e], acc[2][e], acc[3][e]};
    }
  }
}
