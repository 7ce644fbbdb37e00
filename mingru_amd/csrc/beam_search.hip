// A beam search's selection over beams and vocabulary, and the reordering of states (gfx950).
//
// beam_select: of the scores s_k + x_kv - log sum_v exp(x_kv) of K beams and V tokens, the W best.
//
// Bound by memory: the logits are read once.  Within a beam the order of the scores is that of
// the logits, so a first launch reads each row in parts, a wave a part, and leaves a part's
// maximum, sum of exponentials and W largest logits; a second one, a workgroup for each search,
// joins a row's sums and ranks the parts' candidates by their scores in fp64.
//
// The W largest (W <= 64) of a stream of keys, in one wave: the best 64 so far lie sorted over
// the lanes.  A key that beats the W-th of them goes to a buffer in LDS; 64 of them are
// sorted and merged (bitonic, over the lanes).  A long row has few such keys: after n of them
// a new one comes with W / n, so that most tiles cost a comparison.  Before the first tile
// nothing is known; the W-th largest of its lanes' maxima is a bound that W keys reach.
// Keys are whole numbers that order as (value, lower index first), no two alike: the result
// does not depend on the order of arrival, and ties fall as they are defined.
//
// reorder_states: rows of up to 32 tensors a launch, in the largest units of 1 to 16 bytes that
// their sizes, strides and pointers allow.
#include "mg_paged.h"

namespace {

// ---- sorted lists over a wave -----------------------------------------------------------
// Orders as (value, lower index first); 0 is below every key.
struct Key32 {
  unsigned long long k;
  __device__ __forceinline__ bool above(const Key32& o) const { return k > o.k; }
  __device__ __forceinline__ Key32 from(int lane) const {
    return Key32{(unsigned long long)__shfl((long long)k, lane)};
  }
};
struct Key64 {
  unsigned long long k;
  unsigned i;  // ~index
  __device__ __forceinline__ bool above(const Key64& o) const {
    return k > o.k || (k == o.k && i > o.i);
  }
  __device__ __forceinline__ Key64 from(int lane) const {
    return Key64{(unsigned long long)__shfl((long long)k, lane), (unsigned)__shfl((int)i, lane)};
  }
};

__device__ __forceinline__ unsigned bs_order(float x) {
  const unsigned u = __float_as_uint(x + 0.f);  // -0 becomes 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float bs_value(unsigned o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ unsigned long long bs_order(double x) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double bs_value(unsigned long long o) {
  return __longlong_as_double((long long)(o >> 63 ? o & ~(1ull << 63) : ~o));
}

__device__ __forceinline__ int bs_lane() { return threadIdx.x & (MG_WAVE - 1); }

// One exchange with lane ^ d: the larger key stays where `up` holds.
template <typename K>
__device__ __forceinline__ void bs_swap(K& x, int d, bool up) {
  const K o = x.from(bs_lane() ^ d);
  x = x.above(o) == up ? x : o;
}
// Falling over the lanes.
template <typename K>
__device__ __forceinline__ void bs_sort(K& x) {
  const int lane = bs_lane();
  for (int n = 2; n <= MG_WAVE; n *= 2)
    for (int d = n / 2; d > 0; d /= 2) bs_swap(x, d, ((lane & d) == 0) == ((lane & n) == 0));
}
// The 64 largest of two falling lists.
template <typename K>
__device__ __forceinline__ void bs_merge(K& best, const K& more) {
  const K o = more.from(MG_WAVE - 1 - bs_lane());
  if (o.above(best)) best = o;
  for (int d = MG_WAVE / 2; d > 0; d /= 2) bs_swap(best, d, (bs_lane() & d) == 0);
}

// The W largest of what is offered.  buffer: 2 * 64 keys of LDS, the wave's own.
template <typename K>
struct Best {
  K best, bar;  // bar: the W-th largest so far, or a bound that W keys reach
  K* buffer;
  int count, W;
  bool bound;  // bar is such a bound: a key like it counts
  __device__ __forceinline__ void init(K* lds, int width) {
    best = K{}, bar = K{}, buffer = lds, count = 0, W = width, bound = false;
  }
  __device__ __forceinline__ void flush() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int lane = bs_lane(), n = count < MG_WAVE ? count : MG_WAVE;
    K x = lane < n ? buffer[lane] : K{};
    bs_sort(x);
    bs_merge(best, x);
    const K last = best.from(W - 1);
    if (last.above(bar) || !bar.above(last)) bar = last, bound = false;
    const K rest = lane < count - n ? buffer[n + lane] : K{};
    __builtin_amdgcn_wave_barrier();
    if (lane < count - n) buffer[lane] = rest;
    count -= n;
  }
  // One key of each lane, K{} for none.
  __device__ __forceinline__ void offer(const K& x) {
    const bool in = x.above(K{}) && (x.above(bar) || (bound && !bar.above(x)));
    const unsigned long long who = __ballot(in);
    if (who == 0) return;
    if (in) buffer[count + __popcll(who & ((1ull << bs_lane()) - 1))] = x;
    count += __popcll(who);
    if (count >= MG_WAVE) flush();
  }
  // A bound from the lanes' largest keys, before anything is offered.
  __device__ __forceinline__ void hint(K x) {
    bs_sort(x);
    bar = x.from(W - 1);
    bound = true;
  }
  __device__ __forceinline__ void finish() {
    while (count) flush();
  }
};

// ---- rows in parts -----------------------------------------------------------------------
struct BsArgs {
  const void* logits;
  const float* scores;
  const unsigned char* finished;  // or null
  int64_t sb, sk;                 // strides of the logits in elements
  int64_t ss[2], fs[2];           // of the scores and of finished
  int64_t B;
  int K, V, W, end;
  int parts, per;                 // of a row; elements of a part, a multiple of a tile's
  float2* stats;                  // (B, K, parts): maximum, sum
  unsigned long long* keys;       // (B, K, parts, W)
  float* out;
  int64_t *parents, *tokens;
  unsigned char* done;            // or null
};

constexpr int BS_NW = 4, BS_NT = BS_NW * MG_WAVE;
constexpr int BS_VECTORS = 4;  // of 16 bytes, of a lane in a tile

__device__ __forceinline__ bool bs_finished(const BsArgs& a, int64_t b, int k) {
  return a.finished && a.finished[b * a.fs[0] + k * a.fs[1]];
}
__device__ __forceinline__ bool bs_finite(float x) { return fabsf(x) < __builtin_inff(); }

template <typename T>
struct BsVec {
  static constexpr int N = 16 / sizeof(T);
};

template <typename T>
__global__ __launch_bounds__(BS_NT) void beam_rows(BsArgs a) {
  constexpr int N = BsVec<T>::N, ALL = N * BS_VECTORS, TILE = ALL * MG_WAVE;
  __shared__ Key32 s_buffer[BS_NW][2 * MG_WAVE];
  const int lane = bs_lane(), wave = (int)mg_uniform(threadIdx.x / MG_WAVE);
  const int64_t id = (int64_t)blockIdx.x * BS_NW + wave;
  const int64_t row = id / a.parts;
  if (row >= a.B * a.K) return;
  const int part = (int)(id - row * a.parts);
  const int64_t b = row / a.K;
  const int k = (int)(row - b * a.K);
  if (bs_finished(a, b, k) || !bs_finite(a.scores[b * a.ss[0] + k * a.ss[1]])) return;
  const T* const x = (const T*)a.logits + b * a.sb + k * a.sk;
  // Vectors start at the 16-byte line that holds the row's first element: what lies before it
  // in that line, and behind the row's end in the last, is in the same page and not used.
  const int skew = (int)(((uintptr_t)x & 15) / sizeof(T));
  const uint4* const lines = (const uint4*)((uintptr_t)x & ~(uintptr_t)15);
  const int all = a.V + skew;  // elements from the first line on
  const int begin = part * a.per, stop = all - begin < a.per ? all : begin + a.per;

  Best<Key32> list;
  list.init(s_buffer[wave], a.W);
  // No maximum is below the lowest number, so that a lane of -inf alone, or without an element,
  // has a sum of 0.
  float top = -3.402823466e38f, sum = 0.f;
  for (int at = begin; at < stop; at += TILE) {
    uint4 raw[BS_VECTORS];
#pragma unroll
    for (int i = 0; i < BS_VECTORS; ++i) {
      const int e = at + (i * MG_WAVE + lane) * N;
      raw[i] = lines[(e < stop ? e : begin) / N];
    }
    float v[ALL];
    float peak = -__builtin_inff();
    const bool whole = at >= skew && at + TILE <= stop;
#pragma unroll
    for (int i = 0; i < BS_VECTORS; ++i) {
      const T* p = (const T*)&raw[i];
#pragma unroll
      for (int j = 0; j < N; ++j) v[i * N + j] = pg_float(p[j]);
    }
    if (!whole) {  // what is not in the row adds nothing
#pragma unroll
      for (int i = 0; i < ALL; ++i) {
        const int e = at + ((i / N) * MG_WAVE + lane) * N + i % N;
        v[i] = e >= skew && e < stop ? v[i] : -__builtin_inff();
      }
    }
#pragma unroll
    for (int i = 0; i < ALL; ++i) peak = fmaxf(peak, v[i]);
    const float next = fmaxf(top, peak);
    sum *= __expf(top - next);
    float add = 0.f;
#pragma unroll
    for (int i = 0; i < ALL; ++i) add += __expf(v[i] - next);
    sum += add;
    top = next;
    auto key = [&](int i) {
      const int e = at + ((i / N) * MG_WAVE + lane) * N + i % N;
      const bool in = e >= skew && e < stop;
      return Key32{in ? (unsigned long long)bs_order(v[i]) << 32 | ~(unsigned)(e - skew) : 0ull};
    };
    if (at == begin) {
      Key32 most = {0};
#pragma unroll
      for (int i = 0; i < ALL; ++i) {
        const Key32 x = key(i);
        most = x.above(most) ? x : most;
      }
      list.hint(most);
    } else if (__ballot(bs_order(peak) >= (unsigned)(list.bar.k >> 32)) == 0) {
      continue;
    }
#pragma unroll
    for (int i = 0; i < ALL; ++i) list.offer(key(i));
  }
  list.finish();
  float m = top;
#pragma unroll
  for (int d = 1; d < MG_WAVE; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
  const float total = mg_group_sum<64>(sum * __expf(top - m));
  if (lane == 0) a.stats[id] = make_float2(m, total);
  if (lane < a.W) a.keys[id * a.W + lane] = list.best.k;
}

// ---- the selection -----------------------------------------------------------------------
constexpr int BS_MAX_K = 256;

template <int NW>
__global__ __launch_bounds__(NW* MG_WAVE) void beam_pick(BsArgs a) {
  __shared__ Key64 s_buffer[NW][2 * MG_WAVE];
  __shared__ double s_norm[BS_MAX_K], s_score[BS_MAX_K];
  __shared__ unsigned char s_kind[BS_MAX_K];
  enum { LIVE = 0, FINISHED = 1, DEAD = 2 };
  const int lane = bs_lane(), wave = (int)mg_uniform(threadIdx.x / MG_WAVE);
  const int64_t b = blockIdx.x;
  for (int k = wave; k < a.K; k += NW) {
    const float score = a.scores[b * a.ss[0] + k * a.ss[1]];
    const bool finite = bs_finite(score), over = bs_finished(a, b, k);
    float m = -__builtin_inff();
    double sum = 0.0;
    if (finite && !over) {
      const float2* st = a.stats + (b * a.K + k) * a.parts;
      for (int i = lane; i < a.parts; i += MG_WAVE) m = fmaxf(m, st[i].x);
#pragma unroll
      for (int d = 1; d < MG_WAVE; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
      for (int i = lane; i < a.parts; i += MG_WAVE) sum += (double)st[i].y * (double)__expf(st[i].x - m);
#pragma unroll
      for (int d = 1; d < MG_WAVE; d *= 2) sum += __shfl_xor(sum, d);
    }
    if (lane == 0) {
      const double norm = (double)m + log(sum);
      s_score[k] = score, s_norm[k] = over ? 0.0 : norm;
      s_kind[k] = !finite ? DEAD : (over ? FINISHED : (fabs(norm) < __builtin_inf() ? LIVE : DEAD));
    }
  }
  __syncthreads();

  Best<Key64> list;
  list.init(s_buffer[wave], a.W);
  const int each = a.parts * a.W, all = a.K * each;
  for (int at = wave * MG_WAVE; at < all; at += NW * MG_WAVE) {
    const int n = at + lane;
    Key64 x = {0, 0};
    if (n < all) {
      const int k = n / each, r = n - k * each;
      if (s_kind[k] == LIVE) {
        const unsigned long long key = a.keys[(b * a.K + k) * each + r];
        if (key) {
          const unsigned token = ~(unsigned)key;
          x.k = bs_order(s_score[k] + ((double)bs_value((unsigned)(key >> 32)) - s_norm[k]));
          x.i = ~((unsigned)k * (unsigned)a.V + token);
        }
      } else if (r < a.W) {  // without a part of the row: its end, and the first tokens at -inf
        const bool over = s_kind[k] == FINISHED, first = over && r == 0;
        int token = first ? a.end : r - (over ? 1 : 0);
        if (over && !first && token >= a.end) ++token;
        if (token < a.V) {
          x.k = bs_order(first ? s_score[k] : -__builtin_inf());
          x.i = ~((unsigned)k * (unsigned)a.V + (unsigned)token);
        }
      }
    }
    if (at == wave * MG_WAVE) list.hint(x);
    list.offer(x);
  }
  list.finish();
  // The waves' lists, joined by the first.
  __syncthreads();
  if (lane < a.W) s_buffer[wave][lane] = list.best;
  __syncthreads();
  if (wave != 0) return;
  for (int w = 1; w < NW; ++w) bs_merge(list.best, lane < a.W ? s_buffer[w][lane] : Key64{0, 0});
  if (lane < a.W) {
    const unsigned flat = ~list.best.i;
    const int k = (int)(flat / (unsigned)a.V), token = (int)(flat - (unsigned)k * (unsigned)a.V);
    const int64_t n = b * a.W + lane;
    a.out[n] = (float)bs_value(list.best.k);
    a.parents[n] = k, a.tokens[n] = token;
    if (a.done) a.done[n] = token == a.end || bs_finished(a, b, k);
  }
}

// Waves of a row: enough to fill the chip's 256 CUs with 8 waves each, no less than a tile each.
int bs_parts(int64_t rows, int V, int tile) {
  int64_t want = (2048 + rows - 1) / rows;
  const int64_t most = ((int64_t)V + 8 + tile - 1) / tile;
  return (int)(want < most ? want : most);
}
int bs_tile(int dtype) { return (dtype == 0 ? 4 : 8) * BS_VECTORS * MG_WAVE; }
bool bs_ok(int dtype, int64_t B, int64_t K, int64_t V, int W) {
  return dtype >= 0 && dtype <= 2 && B >= 1 && K >= 1 && V >= 1 && K <= BS_MAX_K && W >= 1 &&
         W <= MG_WAVE && V < 1ll << 30 && K * V < 1ll << 31 && W <= K * V && B < 1ll << 22 &&
         B * K < 1ll << 22;
}

// ---- rows of states ------------------------------------------------------------------------
constexpr int RO_MOST = 32, RO_NT = 256, RO_UNITS = 4;  // units of a thread

struct RoTensor {
  const unsigned char* src;
  unsigned char* dst;
  int64_t stride;     // bytes between rows of src
  int64_t units;      // of a row
  int64_t first;      // workgroup of this tensor
};
struct RoArgs {
  RoTensor t[RO_MOST];
  unsigned char shift[RO_MOST];  // log2 of a unit's bytes
  Ints parents;
  int64_t ps[2];
  int64_t K;
  unsigned W;
  int64_t rows;  // B W
  int count;
};

template <typename U>
__device__ __forceinline__ void ro_copy(const RoTensor& t, const RoArgs& a, int64_t first) {
  const int64_t all = a.rows * t.units;
  const int64_t row0 = first / t.units, in0 = first - row0 * t.units;
  U v[RO_UNITS];
#pragma unroll
  for (int i = 0; i < RO_UNITS; ++i) {
    const int64_t n = first + i * RO_NT + threadIdx.x;
    v[i] = U{};
    if (n < all) {
      int64_t in = in0 + i * RO_NT + threadIdx.x, row = row0;
      if (in >= t.units) {
        // At most RO_UNITS RO_NT past a row's start, or the row is longer and this the next.
        if (t.units > RO_UNITS * RO_NT) {
          in -= t.units, row += 1;
        } else {
          const unsigned q = (unsigned)in / (unsigned)t.units;
          in -= (int64_t)q * t.units, row += q;
        }
      }
      const unsigned b = (unsigned)row / a.W, w = (unsigned)row - b * a.W;
      const int64_t parent = a.parents[b * a.ps[0] + w * a.ps[1]];
      if (parent >= 0 && parent < a.K)
        v[i] = *(const U*)(t.src + (b * a.K + parent) * t.stride + in * (int64_t)sizeof(U));
    }
  }
#pragma unroll
  for (int i = 0; i < RO_UNITS; ++i) {
    const int64_t n = first + i * RO_NT + threadIdx.x;
    if (n < all) *(U*)(t.dst + n * (int64_t)sizeof(U)) = v[i];
  }
}

__global__ __launch_bounds__(RO_NT) void reorder_rows(RoArgs a) {
  int i = 0;
  while (i + 1 < a.count && (int64_t)blockIdx.x >= a.t[i + 1].first) ++i;
  const RoTensor t = a.t[i];
  const int64_t first = ((int64_t)blockIdx.x - t.first) * (RO_NT * RO_UNITS);
  switch (a.shift[i]) {
    case 4: ro_copy<u32x4>(t, a, first); break;
    case 3: ro_copy<u32x2>(t, a, first); break;
    case 2: ro_copy<unsigned>(t, a, first); break;
    case 1: ro_copy<u16>(t, a, first); break;
    default: ro_copy<unsigned char>(t, a, first);
  }
}

}  // namespace

extern "C" {

size_t mg_beam_select_workspace_bytes(int dtype, int64_t B, int64_t K, int64_t V, int W) {
  if (!bs_ok(dtype, B, K, V, W)) return 0;
  const size_t parts = (size_t)B * K * bs_parts(B * K, (int)V, bs_tile(dtype));
  return parts * (sizeof(float2) + W * sizeof(unsigned long long));
}

int mg_beam_select(int dtype, const void* logits, const float* scores, const void* finished,
                   const int64_t* strides, int64_t end, float* out, int64_t* parents,
                   int64_t* tokens, void* done, int64_t B, int64_t K, int64_t V, int W, void* ws,
                   size_t ws_bytes, hipStream_t stream) {
  if (!logits || !scores || !strides || !out || !parents || !tokens || !ws ||
      !bs_ok(dtype, B, K, V, W) || end >= V || (end < 0 && (finished || done)))
    return MG_ERR_ARG;
  if (ws_bytes < mg_beam_select_workspace_bytes(dtype, B, K, V, W)) return MG_ERR_WORKSPACE;
  BsArgs a = {};
  a.logits = logits, a.scores = scores, a.finished = (const unsigned char*)finished;
  a.sb = strides[0], a.sk = strides[1];
  for (int i = 0; i < 2; ++i) a.ss[i] = strides[2 + i], a.fs[i] = strides[4 + i];
  a.B = B, a.K = (int)K, a.V = (int)V, a.W = W, a.end = (int)end;
  const int tile = bs_tile(dtype);
  a.parts = bs_parts(B * K, (int)V, tile);
  const int64_t per = (V + 8 + a.parts - 1) / a.parts;
  a.per = (int)((per + tile - 1) / tile * tile);
  a.parts = (int)((V + 8 + a.per - 1) / a.per);
  a.keys = (unsigned long long*)ws;
  a.stats = (float2*)(a.keys + B * K * a.parts * W);
  a.out = out, a.parents = parents, a.tokens = tokens, a.done = (unsigned char*)done;
  const dim3 grid((unsigned)((B * K * a.parts + BS_NW - 1) / BS_NW)), nt(BS_NT);
  if (dtype == 0) hipLaunchKernelGGL(beam_rows<float>, grid, nt, 0, stream, a);
  else if (dtype == 1) hipLaunchKernelGGL(beam_rows<Bf16>, grid, nt, 0, stream, a);
  else hipLaunchKernelGGL(beam_rows<Fp16>, grid, nt, 0, stream, a);
  if (hipGetLastError() != hipSuccess) return MG_ERR_LAUNCH;
  hipLaunchKernelGGL(beam_pick<4>, dim3((unsigned)B), dim3(4 * MG_WAVE), 0, stream, a);
  return hipGetLastError() == hipSuccess ? MG_OK : MG_ERR_LAUNCH;
}

int mg_reorder_rows(int count, const void* const* src, void* const* dst, const int64_t* strides,
                    const int64_t* bytes, int wide, const void* parents, int64_t pb, int64_t pw,
                    int64_t B, int64_t K, int64_t W, hipStream_t stream) {
  if (count < 1 || !src || !dst || !strides || !bytes || (wide & ~1) || !parents || B < 1 ||
      K < 1 || W < 1 || W >= 1ll << 31 || B >= 1ll << 31 || B * W >= 1ll << 31 ||
      K >= 1ll << 31)
    return MG_ERR_ARG;
  for (int i = 0; i < count; ++i)
    if (!src[i] || !dst[i] || bytes[i] < 1 || bytes[i] >= 1ll << 40) return MG_ERR_ARG;
  for (int at = 0; at < count; at += RO_MOST) {
    RoArgs a = {};
    a.parents = Ints{parents, wide}, a.ps[0] = pb, a.ps[1] = pw;
    a.K = K, a.W = (unsigned)W, a.rows = B * W;
    a.count = count - at < RO_MOST ? count - at : RO_MOST;
    int64_t groups = 0;
    for (int i = 0; i < a.count; ++i) {
      RoTensor& t = a.t[i];
      t.src = (const unsigned char*)src[at + i], t.dst = (unsigned char*)dst[at + i];
      t.stride = strides[at + i], t.first = groups;
      const uint64_t odd = (uint64_t)(uintptr_t)t.src | (uint64_t)(uintptr_t)t.dst |
                           (uint64_t)t.stride | (uint64_t)bytes[at + i];
      int shift = 0;
      while (shift < 4 && !(odd >> shift & 1)) ++shift;
      a.shift[i] = (unsigned char)shift;
      t.units = bytes[at + i] >> shift;
      groups += (a.rows * t.units + RO_NT * RO_UNITS - 1) / (RO_NT * RO_UNITS);
      if (groups >= 1ll << 24) return MG_ERR_TOO_LARGE;  // 2^32 threads
    }
    hipLaunchKernelGGL(reorder_rows, dim3((unsigned)groups), dim3(RO_NT), 0, stream, a);
    if (hipGetLastError() != hipSuccess) return MG_ERR_LAUNCH;
  }
  return MG_OK;
}

}  // extern "C"
