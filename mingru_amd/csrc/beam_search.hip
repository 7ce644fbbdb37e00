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
// the lanes.  Of the keys that a lane each offers, those that beat the W-th of them are put in
// one by one where they are few, or sorted and merged (bitonic, over the lanes).  A long row has
// few such keys: after n of them a new one comes with W / n, so that most elements cost a
// comparison of values.  A first bar is the W-th of the lanes' largest values of the first tile.
// Lanes exchange keys by row operations and swaps of half rows, without LDS.
// Keys are whole numbers that order as (value, lower index first), no two alike: the result
// does not depend on the order of arrival, and ties fall as they are defined.
//
// 64 x 8 rows of 50257 in bf16, a fifth of them not read: 17 us for 41 MB and 6 for the selection.
// What is left above the memory's 8 is the exponentials and comparisons (the vector units issue
// half of the time) and a wave's two sorts, each a chain of 21 exchanges.
//
// reorder_states: rows of up to 32 tensors a launch, in vectors of 16 bytes of the output, whose rows
// follow one another.  A vector lies in one row, read from wherever that starts, or holds the end of
// one and the start of the next, read byte by byte; rows of fewer bytes go in the largest units
// that sizes, strides and pointers allow.
#include "mg_paged.h"

namespace {

// ---- sorted lists over a wave -----------------------------------------------------------
__device__ __forceinline__ int bs_lane() { return threadIdx.x & (MG_WAVE - 1); }

// x of lane ^ D.
template <int CTRL>
__device__ __forceinline__ unsigned bs_dpp(unsigned x) {
  return (unsigned)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xf, 0xf, false);
}
template <int D>
__device__ __forceinline__ unsigned bs_xor(unsigned x) {
  if constexpr (D == 1) {
    return bs_dpp<0xB1>(x);  // quad_perm 1, 0, 3, 2
  } else if constexpr (D == 2) {
    return bs_dpp<0x4E>(x);  // quad_perm 2, 3, 0, 1
  } else if constexpr (D == 4) {
    return bs_dpp<0x1B>(bs_dpp<0x141>(x));  // lane ^ 7 (row_half_mirror), then ^ 3
  } else if constexpr (D == 8) {
    return bs_dpp<0x128>(x);  // row_ror:8
  } else if constexpr (D == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return bs_lane() & 16 ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return bs_lane() & 32 ? r[0] : r[1];
  }
}
// x of lane ^ 63.
__device__ __forceinline__ unsigned bs_mirror(unsigned x) {
  return bs_xor<32>(bs_xor<16>(bs_dpp<0x140>(x)));  // row_mirror: lane ^ 15
}
__device__ __forceinline__ unsigned bs_read(unsigned x, int lane) {
  return (unsigned)__builtin_amdgcn_readlane((int)x, lane);
}
__device__ __forceinline__ unsigned bs_prev(unsigned x) {  // of the lane before; 0 in lane 0
  return __float_as_uint(mg_wave_prev(__uint_as_float(x)));
}

// A key orders as (value, lower index first); 0 is below every key.  Key32's value is of 32
// bits, above its inverted index; Key64's of 64.  Words by name, not in an array: a choice
// between two arrays' elements becomes one between their addresses, in memory.
__device__ __forceinline__ unsigned long long bs_join(unsigned hi, unsigned lo) {
  return (unsigned long long)hi << 32 | lo;
}
struct Key32 {
  unsigned index, value;
  __device__ __forceinline__ unsigned long long all() const { return bs_join(value, index); }
  __device__ __forceinline__ bool above(Key32 o) const { return all() > o.all(); }
  template <typename F>
  __device__ __forceinline__ Key32 map(F&& f) const {
    return Key32{f(index), f(value)};
  }
  __device__ __forceinline__ Key32 pick(bool first, Key32 o) const {
    return Key32{first ? index : o.index, first ? value : o.value};
  }
};
struct Value32 {  // no index: for a bar
  unsigned value;
  __device__ __forceinline__ bool above(Value32 o) const { return value > o.value; }
  template <typename F>
  __device__ __forceinline__ Value32 map(F&& f) const {
    return Value32{f(value)};
  }
  __device__ __forceinline__ Value32 pick(bool first, Value32 o) const {
    return Value32{first ? value : o.value};
  }
};
struct Key64 {
  unsigned index, lo, hi;
  __device__ __forceinline__ unsigned long long value() const { return bs_join(hi, lo); }
  __device__ __forceinline__ bool above(Key64 o) const {
    return value() > o.value() || (value() == o.value() && index > o.index);
  }
  template <typename F>
  __device__ __forceinline__ Key64 map(F&& f) const {
    return Key64{f(index), f(lo), f(hi)};
  }
  __device__ __forceinline__ Key64 pick(bool first, Key64 o) const {
    return Key64{first ? index : o.index, first ? lo : o.lo, first ? hi : o.hi};
  }
};
template <typename K>
__device__ __forceinline__ K bs_from(K x, int lane) {  // the same lane for all
  return x.map([=](unsigned w) { return bs_read(w, lane); });
}

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

// One exchange with lane ^ D: the larger key stays where `up` holds.
template <int D, typename K>
__device__ __forceinline__ K bs_swap(K x, bool up) {
  const K o = x.map([](unsigned w) { return bs_xor<D>(w); });
  return x.pick(x.above(o) == up, o);
}
// A bitonic row of 2 D lanes becomes falling (up) or rising.
template <int D, typename K>
__device__ __forceinline__ K bs_settle(K x, bool up) {
  x = bs_swap<D>(x, ((bs_lane() & D) == 0) == up);
  if constexpr (D > 1) x = bs_settle<D / 2>(x, up);
  return x;
}
// Falling over the lanes.
template <typename K>
__device__ __forceinline__ K bs_sort(K x) {
  const int lane = bs_lane();
  x = bs_settle<1>(x, (lane & 2) == 0);
  x = bs_settle<2>(x, (lane & 4) == 0);
  x = bs_settle<4>(x, (lane & 8) == 0);
  x = bs_settle<8>(x, (lane & 16) == 0);
  x = bs_settle<16>(x, (lane & 32) == 0);
  return bs_settle<32>(x, true);
}
// The 64 largest of two falling lists.
template <typename K>
__device__ __forceinline__ K bs_merge(K best, K more) {
  const K o = more.map([](unsigned w) { return bs_mirror(w); });
  return bs_settle<32>(o.pick(o.above(best), best), true);
}

// The W largest of what is offered.
template <typename K>
struct Best {
  K best, bar;  // falling over the lanes; the W-th of them, or floor where that is above
  K floor;      // a key that W of all keys reach, here or elsewhere
  int last;     // W - 1
  __device__ __forceinline__ void settle() {
    const K x = bs_from(best, last);
    bar = floor.pick(floor.above(x), x);
  }
  __device__ __forceinline__ void start(int W) { best = K{}, bar = K{}, floor = K{}, last = W - 1; }
  // One key of each lane, 0 for none.
  __device__ __forceinline__ void offer(K x) {
    const bool in = x.above(bar);
    unsigned long long who = __ballot(in);
    if (who == 0) return;
    // Where a sort's 27 exchanges cost less.
    if (__popcll(who) > 8) {
      best = bs_merge(best, bs_sort(x.pick(in, K{})));
    } else {
      do {
        const K one = bs_from(x, __ffsll(who) - 1);
        who &= who - 1;
        const int at = __popcll(__ballot(best.above(one)));
        const K up = best.map([](unsigned w) { return bs_prev(w); });
        best = best.pick(bs_lane() < at, one.pick(bs_lane() == at, up));
      } while (who);
    }
    settle();
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
  unsigned long long* keys;       // (B, W, K, parts)
  float* out;
  int64_t *parents, *tokens;
  unsigned char* done;            // or null
};

constexpr int BS_NW = 4, BS_NT = BS_NW * MG_WAVE;
constexpr int BS_EACH = 32;    // elements of a lane in a tile
constexpr int BS_HITS = 512;   // elements that are kept to be offered
constexpr int BS_READY = 32;   // more are offered

__device__ __forceinline__ bool bs_finished(const BsArgs& a, int64_t b, int k) {
  return a.finished && a.finished[b * a.fs[0] + k * a.fs[1]];
}
__device__ __forceinline__ float bs_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }
__device__ __forceinline__ bool bs_finite(float x) { return fabsf(x) < __builtin_inff(); }

template <typename T>
struct BsVec {
  static constexpr int N = 16 / sizeof(T);
};

template <typename T>
__global__ __launch_bounds__(BS_NT, 4) void beam_rows(BsArgs a) {
  constexpr int N = BsVec<T>::N, VECTORS = BS_EACH / N, ALL = BS_EACH, TILE = ALL * MG_WAVE;
  __shared__ int s_place[BS_NW][BS_HITS];  // elements that reach the bar
  const int lane = bs_lane(), wave = (int)mg_uniform(threadIdx.x / MG_WAVE);
  const int64_t id = (int64_t)blockIdx.x * BS_NW + wave;
  const int64_t row = id / a.parts;
  if (row >= a.B * a.K) return;
  const int part = (int)(id - row * a.parts);
  const int64_t b = row / a.K;
  const int k = (int)(row - b * a.K);
  const T* const x = (const T*)a.logits + b * a.sb + k * a.sk;
  // Vectors start at the 16-byte line that holds the row's first element: what lies before it
  // in that line, and behind the row's end in the last, is in the same page and not used.
  const int skew = (int)(((uintptr_t)x & 15) / sizeof(T));
  const uint4* const lines = (const uint4*)((uintptr_t)x & ~(uintptr_t)15);
  const int all = a.V + skew;  // elements from the first line on
  const int begin = part * a.per, stop = all - begin < a.per ? all : begin + a.per;

  Best<Key32> list;
  list.start(a.W);
  // No maximum is below the lowest number, so that a lane of -inf alone, or without an element,
  // has a sum of 0.
  float top = -3.402823466e38f, sum = 0.f;
  // A tile ahead; the first is on its way before it is known whether the row counts.
  uint4 raw[VECTORS];
  auto load = [&](int at) {
#pragma unroll
    for (int i = 0; i < VECTORS; ++i) {
      const int e = at + (i * MG_WAVE + lane) * N;
      raw[i] = lines[(e < stop ? e : begin) / N];
    }
  };
  int kept = 0;
  if (begin < stop) load(begin);
  const float score = a.scores[b * a.ss[0] + k * a.ss[1]];
  if (bs_finished(a, b, k) || !bs_finite(score)) return;
  for (int at = begin; at < stop; at += TILE) {
    float v[ALL];
    float peak = -__builtin_inff();
    const bool whole = at >= skew && at + TILE <= stop;
#pragma unroll
    for (int i = 0; i < VECTORS; ++i) {
      const T* p = (const T*)&raw[i];
#pragma unroll
      for (int j = 0; j < N; ++j) v[i * N + j] = pg_float(p[j]);
    }
    load(at + TILE < stop ? at + TILE : begin);
    if (!whole) {  // what is not in the row adds nothing
#pragma unroll
      for (int i = 0; i < ALL; ++i) {
        const int e = at + ((i / N) * MG_WAVE + lane) * N + i % N;
        v[i] = e >= skew && e < stop ? v[i] : -__builtin_inff();
      }
    }
    float peaks[VECTORS];
#pragma unroll
    for (int i = 0; i < VECTORS; ++i) {
      peaks[i] = v[i * N];
#pragma unroll
      for (int j = 1; j < N; ++j) peaks[i] = fmaxf(peaks[i], v[i * N + j]);
      peak = fmaxf(peak, peaks[i]);
    }
    const float next = fmaxf(top, peak);
    sum *= bs_exp(top - next);
    float add[2] = {0.f, 0.f};
    if (__ballot(!(fabsf(next) < 1048576.f)) == 0) {
      // exp(v - next) as 2^(v L - c), L = log2 e, one operation less: c is next L rounded, and what
      // that rounds off, r, the same for all of them, is put back once.  Below 2^20 it is 2^-4 at
      // most; without a bound it would grow with next until 2^r is out of range.
      const float c = next * 1.44269504f, r = __builtin_fmaf(next, 1.44269504f, -c);
#pragma unroll
      for (int i = 0; i < ALL; ++i)
        add[i & 1] += __builtin_amdgcn_exp2f(__builtin_fmaf(v[i], 1.44269504f, -c));
      sum += (add[0] + add[1]) * __builtin_amdgcn_exp2f(-r);
    } else {
#pragma unroll
      for (int i = 0; i < ALL; ++i) add[i & 1] += bs_exp(v[i] - next);
      sum += add[0] + add[1];
    }
    top = next;
    if (at == begin) {
      const Value32 bar = bs_from(bs_sort(Value32{bs_order(peak)}), a.W - 1);
      list.floor = Key32{0, bar.value};  // below every key of that value
      list.settle();
    }
    const float bar = bs_value(list.bar.value);
    // A bit for each element that does; then each lane's first one, its second, and so on go to the
    // list.  (A test of the whole wave for each element is a chain of some thirty round trips
    // between the vector and the scalar unit: 8 us of 28 at 512 rows of 50257 in bf16.)
    int hits = kept;
    unsigned bits = 0;
#pragma unroll
    for (int g = 0; g < VECTORS; ++g) {
      if (__ballot(peaks[g] >= bar) == 0) continue;
#pragma unroll
      for (int i = g * N; i < g * N + N; ++i) bits |= v[i] >= bar ? 1u << i : 0u;
    }
    for (unsigned long long who; (who = __ballot(bits != 0)) != 0; bits &= bits - 1) {
      const int i = __ffs(bits) - 1, to = hits + (int)__builtin_amdgcn_mbcnt_hi(
          (unsigned)(who >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)who, 0));
      if (bits != 0 && to < BS_HITS)
        s_place[wave][to] = at + (i / N * MG_WAVE + lane) * N + i % N;
      hits += __popcll(who);
    }
    // They are offered when there are many, or no more to come.  Where a tile has more than there
    // is room for (rows full of ties, rising rows), those of the tiles before, then the whole tile.
    const bool again = hits > BS_HITS;
    const int ready = again ? kept : (hits > BS_READY || at + TILE >= stop ? hits : 0);
    kept = ready || again ? 0 : hits;
    const int chunks = (ready + MG_WAVE - 1) / MG_WAVE, every = chunks + (again ? ALL : 0);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    for (int n = 0; n < every; ++n) {
      const bool from = n < chunks;
      const int i = n * MG_WAVE + lane;
      const int e = from ? s_place[wave][i < ready ? i : 0] : at + i - chunks * MG_WAVE;
      const bool in = (!from || i < ready) && e >= skew && e < stop;
      const float value = pg_float(x[in ? e - skew : 0]);
      list.offer(Key32{in ? ~(unsigned)(e - skew) : 0u, in ? bs_order(value) : 0u});
    }
    __builtin_amdgcn_wave_barrier();
  }
  float m = top;
#pragma unroll
  for (int d = 1; d < MG_WAVE; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
  const float total = mg_group_sum<64>(sum * bs_exp(top - m));
  if (lane == 0) a.stats[id] = make_float2(m, total);
  if (lane < a.W) {
    const int64_t lists = (int64_t)a.K * a.parts;
    a.keys[(b * a.W + lane) * lists + (id - b * lists)] = begin < stop ? list.best.all() : 0ull;
  }
}

// ---- the selection -----------------------------------------------------------------------
constexpr int BS_MAX_K = 256;

__device__ __forceinline__ double bs_row_sum(double x) {  // over 16 lanes
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(x);
    unsigned lo = (unsigned)u, hi = (unsigned)(u >> 32);
    if (i == 0) lo = bs_xor<1>(lo), hi = bs_xor<1>(hi);
    else if (i == 1) lo = bs_xor<2>(lo), hi = bs_xor<2>(hi);
    else if (i == 2) lo = bs_xor<4>(lo), hi = bs_xor<4>(hi);
    else lo = bs_xor<8>(lo), hi = bs_xor<8>(hi);
    x += __longlong_as_double((long long)((unsigned long long)hi << 32 | lo));
  }
  return x;
}

template <int NW>
__global__ __launch_bounds__(NW* MG_WAVE) void beam_pick(BsArgs a) {
  __shared__ Key64 s_list[NW / 2][MG_WAVE], s_bar;
  __shared__ double s_log[BS_MAX_K], s_score[BS_MAX_K];  // of the sum over exp(x - top)
  __shared__ float s_top[BS_MAX_K];
  __shared__ unsigned char s_kind[BS_MAX_K];
  enum { LIVE = 0, FINISHED = 1, DEAD = 2 };
  const int lane = bs_lane(), wave = (int)mg_uniform(threadIdx.x / MG_WAVE);
  const int64_t b = blockIdx.x;
  // Sixteen lanes a row.
  for (int k0 = 0; k0 < a.K; k0 += NW * 4) {
    const int k = k0 + (int)threadIdx.x / 16, in = threadIdx.x & 15;
    const int at = k < a.K ? k : a.K - 1;
    const float score = a.scores[b * a.ss[0] + at * a.ss[1]];
    const bool finite = bs_finite(score), over = bs_finished(a, b, at);
    const float2* st = a.stats + (b * a.K + at) * a.parts;
    float m = -__builtin_inff();
    double sum = 0.0;
    if (finite && !over) {  // written by the first launch
      for (int i = in; i < a.parts; i += 16) m = fmaxf(m, st[i].x);
      m = fmaxf(m, mg_row_ror<8>(m));
      m = fmaxf(m, mg_row_ror<4>(m));
      m = fmaxf(m, mg_row_ror<2>(m));
      m = fmaxf(m, mg_row_ror<1>(m));
      for (int i = in; i < a.parts; i += 16) sum += (double)st[i].y * (double)bs_exp(st[i].x - m);
      sum = bs_row_sum(sum);
    }
    if (in == 0 && k < a.K) {
      const double part = log(sum);
      const bool live = bs_finite(m) && fabs(part) < __builtin_inf();
      s_score[k] = score, s_top[k] = m, s_log[k] = part;
      s_kind[k] = !finite ? DEAD : (over ? FINISHED : (live ? LIVE : DEAD));
    }
  }
  __syncthreads();

  Best<Key64> list;
  // Every part's first candidates come before any part's second ones, so that the first ones that
  // are looked at set a high bar.
  const int lists = a.K * a.parts, all = lists * a.W;
  auto key = [&](double score, unsigned index) {
    const unsigned long long o = bs_order(score);
    return Key64{~index, (unsigned)o, (unsigned)(o >> 32)};
  };
  const unsigned long long* const keys = a.keys + b * all;
  auto raw = [&](int n) { return keys[n < all ? n : 0]; };
  auto candidate = [&](int n, unsigned long long from) {
    Key64 x = {};
    if (n < all) {
      const int r = n / lists, at = n - r * lists, k = at / a.parts;
      if (s_kind[k] == LIVE) {
        if (from)
          // The difference first: a large top would swallow the logarithm.
          x = key(s_score[k] + ((double)bs_value((unsigned)(from >> 32)) - (double)s_top[k] - s_log[k]),
                  (unsigned)k * (unsigned)a.V + ~(unsigned)from);
      } else if (at == k * a.parts) {  // in place of its parts: its end, and the first tokens at -inf
        const bool over = s_kind[k] == FINISHED, first = over && r == 0;
        int token = first ? a.end : r - (over ? 1 : 0);
        if (over && !first && token >= a.end) ++token;
        if (token < a.V)
          x = key(first ? s_score[k] : -__builtin_inf(), (unsigned)k * (unsigned)a.V + (unsigned)token);
      }
    }
    return x;
  };
  // A bar that W candidates reach: of 64 parts' first ones, all over the beams, the W-th.  The
  // candidates that reach it are few more than W.
  int at = wave * MG_WAVE;
  unsigned long long next = raw(at + lane);
  if (wave == 0) {
    const int n = lists > MG_WAVE ? (int)((int64_t)lane * lists / MG_WAVE) : lane;
    const Key64 x = bs_sort(n < all ? candidate(n, raw(n)) : Key64{});
    const Key64 bar = bs_from(x, a.W - 1);
    if (lane == 0) s_bar = bar;
  }
  __syncthreads();
  // Just below that candidate: the inverted index of a key is above 0.
  list.start(a.W);
  list.floor = s_bar;
  if (list.floor.above(Key64{})) list.floor.index -= 1;
  list.settle();
  for (; at < all; at += NW * MG_WAVE) {
    const unsigned long long now = next;
    next = raw(at + NW * MG_WAVE + lane);
    list.offer(candidate(at + lane, now));
  }
  // The waves' lists, by halves.
#pragma unroll
  for (int half = NW / 2; half > 0; half /= 2) {
    if (wave >= half && wave < 2 * half) s_list[wave - half][lane] = list.best;
    __syncthreads();
    if (wave < half) list.best = bs_merge(list.best, s_list[wave][lane]);
    __syncthreads();
  }
  if (wave == 0 && lane < a.W) {
    const unsigned flat = ~list.best.index;
    const int k = (int)(flat / (unsigned)a.V), token = (int)(flat - (unsigned)k * (unsigned)a.V);
    const int64_t n = b * a.W + lane;
    a.out[n] = (float)bs_value(list.best.value());
    a.parents[n] = k, a.tokens[n] = token;
    if (a.done) a.done[n] = token == a.end || bs_finished(a, b, k);
  }
}

// Waves of a row: two for each of the chip's 1024 vector units over all rows, none with less than
// a tile.  (64 x 8 rows of 50257 in bf16, both launches in a graph: 24.6 us; four for each, with
// more first tiles and candidates, 25.8, one 33.  16 x 16 of 32771 in fp32, 32 wide: 32, four 38.)
int bs_parts(int64_t rows, int V, int tile) {
  const int64_t want = (2048 + rows - 1) / rows;
  const int64_t most = ((int64_t)V + 8 + tile - 1) / tile;
  return (int)(want < most ? want : most);
}
constexpr int BS_TILE = BS_EACH * MG_WAVE;
bool bs_ok(int dtype, int64_t B, int64_t K, int64_t V, int W) {
  return dtype >= 0 && dtype <= 2 && B >= 1 && K >= 1 && V >= 1 && K <= BS_MAX_K && W >= 1 &&
         W <= MG_WAVE && V < 1ll << 30 && K * V < 1ll << 31 && W <= K * V && B < 1ll << 22 &&
         B * K < 1ll << 22;
}

// ---- rows of states ------------------------------------------------------------------------
// Units of a thread: 8 layers of 128 rows of 512 KB took 166 us, with four 176, with eight 386.
constexpr int RO_MOST = 32, RO_NT = 256, RO_UNITS = 2;

struct RoTensor {
  const unsigned char* src;
  unsigned char* dst;
  int64_t stride;     // bytes between rows of src
  int64_t units;      // of a row
};
struct RoArgs {
  unsigned first[RO_MOST];  // workgroup of each tensor; those past the last are never reached
  RoTensor t[RO_MOST];
  unsigned char shift[RO_MOST];  // log2 of a unit's bytes
  Ints parents;
  int64_t ps[2];
  int64_t K;
  unsigned W;
  int64_t rows;  // B W
  int count;
  int chunks;    // of a workgroup
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
    if (n < all) __builtin_nontemporal_store(v[i], (U*)(t.dst + n * (int64_t)sizeof(U)));
  }
}

typedef u32x4 u32x4_any __attribute__((aligned(1)));

// The same with vectors that hold 16 bytes of the rows one after another, each of 16 or more (units:
// bytes of a row).
__device__ __forceinline__ void ro_across(const RoTensor& t, const RoArgs& a, int64_t first) {
  const int64_t all = a.rows * t.units, begin = first * 16;
  const int64_t row0 = begin / t.units, in0 = begin - row0 * t.units;
  auto source = [&](int64_t row) -> const unsigned char* {  // null: 0
    const unsigned b = (unsigned)row / a.W, w = (unsigned)row - b * a.W;
    const int64_t parent = a.parents[b * a.ps[0] + w * a.ps[1]];
    return parent >= 0 && parent < a.K ? t.src + (b * a.K + parent) * t.stride : nullptr;
  };
#pragma unroll
  for (int i = 0; i < RO_UNITS; ++i) {
    const int64_t n = begin + (int64_t)(i * RO_NT + threadIdx.x) * 16;
    if (n >= all) continue;
    int64_t in = in0 + (i * RO_NT + threadIdx.x) * 16, row = row0;
    if (in >= t.units) {
      if (t.units > RO_UNITS * RO_NT * 16) {
        in -= t.units, row += 1;
      } else {
        const unsigned q = (unsigned)in / (unsigned)t.units;
        in -= (int64_t)q * t.units, row += q;
      }
    }
    const unsigned char* src = source(row);
    if (in + 16 <= t.units) {
      u32x4 v = {0, 0, 0, 0};
      if (src) v = *(const u32x4_any*)(src + in);
      __builtin_nontemporal_store(v, (u32x4*)(t.dst + n));
      continue;
    }
    // Every byte's load under no condition, so that they are on their way together.
    const int end = all - n < 16 ? (int)(all - n) : 16, here = (int)(t.units - in);
    const unsigned char* const then = here < end ? source(row + 1) : src;
    const unsigned char* const some = src ? src : t.src;
    unsigned w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const unsigned char* from = e < here ? src : then;
      from = e < end && from ? from + (e < here ? in + e : e - here) : nullptr;
      const unsigned byte = *(from ? from : some);
      w[e / 4] |= (from ? byte : 0u) << e % 4 * 8;
    }
    if (end == 16) {
      *(u32x4*)(t.dst + n) = u32x4{w[0], w[1], w[2], w[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 15; ++e)
        if (e < end) t.dst[n + e] = (unsigned char)(w[e / 4] >> e % 4 * 8);
    }
  }
}

// ACROSS: vectors that rows need not end at; a kernel of its own, whose registers and instructions
// the other would pay for (8 layers of 128 rows of 512 KB: 166 us apart, 177 in one).
template <bool ACROSS>
__global__ __launch_bounds__(RO_NT) void reorder_rows(RoArgs a) {
  int i = -1;
#pragma unroll
  for (int j = 0; j < RO_MOST; ++j) i += blockIdx.x >= a.first[j] ? 1 : 0;
  const RoTensor t = a.t[i];
  const int64_t first = (int64_t)(blockIdx.x - a.first[i]) * a.chunks * (RO_NT * RO_UNITS);
  const int shift = a.shift[i];
  for (int c = 0; c < a.chunks; ++c) {
    const int64_t at = first + (int64_t)c * (RO_NT * RO_UNITS);
    if constexpr (ACROSS) {
      ro_across(t, a, at);
    } else {
      switch (shift) {
        case 4: ro_copy<u32x4>(t, a, at); break;
        case 3: ro_copy<u32x2>(t, a, at); break;
        case 2: ro_copy<unsigned>(t, a, at); break;
        case 1: ro_copy<u16>(t, a, at); break;
        default: ro_copy<unsigned char>(t, a, at);
      }
    }
  }
}

}  // namespace

extern "C" {

size_t mg_beam_select_workspace_bytes(int dtype, int64_t B, int64_t K, int64_t V, int W) {
  if (!bs_ok(dtype, B, K, V, W)) return 0;
  const size_t parts = (size_t)B * K * bs_parts(B * K, (int)V, BS_TILE);
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
  const int tile = BS_TILE;
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
  // Eight waves where four would have more than two rounds of candidates: 8 x 8 beams of 31633 take
  // 13.9 us with both launches, with four 14.5; 16 x 16 of 32771, 32 wide, 31.2, four 32.8, sixteen
  // 31.9.
  if (K * a.parts * W <= 2 * 4 * MG_WAVE)
    hipLaunchKernelGGL(beam_pick<4>, dim3((unsigned)B), dim3(4 * MG_WAVE), 0, stream, a);
  else
    hipLaunchKernelGGL(beam_pick<8>, dim3((unsigned)B), dim3(8 * MG_WAVE), 0, stream, a);
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
  // How a tensor's rows go: log2 of a unit's bytes, or across the rows' ends.  The latter where few
  // vectors hold an end: rows of 19137 elements of 2 bytes take 23 us in place of 71 (6 layers of
  // 256 rows), rows of 36 bytes 10 in place of 7.
  auto shift_of = [&](int i) {
    const uint64_t odd = (uint64_t)(uintptr_t)src[i] | (uint64_t)(uintptr_t)dst[i] |
                         (uint64_t)strides[i] | (uint64_t)bytes[i];
    int shift = 0;
    while (shift < 4 && !(odd >> shift & 1)) ++shift;
    return shift;
  };
  auto across_of = [&](int i) {
    return shift_of(i) < 4 && bytes[i] >= 256 && ((uintptr_t)dst[i] & 15) == 0;
  };
  auto units_of = [&](int i) {
    return across_of(i) ? (B * W * bytes[i] + 15) / 16 : B * W * (bytes[i] >> shift_of(i));
  };
  int64_t units = 0;
  for (int i = 0; i < count; ++i) {
    if (bytes[i] >= (1ll << 62) / (B * W)) return MG_ERR_TOO_LARGE;
    units += units_of(i) + RO_NT * RO_UNITS;
    if (units >= (int64_t)(RO_NT * RO_UNITS) << 24) return MG_ERR_TOO_LARGE;  // 2^32 threads
  }
  // Two chunks of a workgroup where they are many: its start costs less (168 us in place of 177 at
  // 537 MB), one where they are few.
  const int chunks = units >= 8ll << 20 ? 2 : 1;
  for (int across = 0; across < 2; ++across) {
    RoArgs a = {};
    a.parents = Ints{parents, wide}, a.ps[0] = pb, a.ps[1] = pw;
    a.K = K, a.W = (unsigned)W, a.rows = B * W;
    a.chunks = chunks;
    int64_t groups = 0;
    for (int i = 0; i < count; ++i) {
      if (across_of(i) == (across != 0)) {
        RoTensor& t = a.t[a.count];
        t.src = (const unsigned char*)src[i], t.dst = (unsigned char*)dst[i], t.stride = strides[i];
        t.units = across ? bytes[i] : bytes[i] >> shift_of(i);
        a.shift[a.count] = (unsigned char)shift_of(i);
        a.first[a.count++] = (unsigned)groups;
        const int64_t each = RO_NT * RO_UNITS * chunks;
        groups += (units_of(i) + each - 1) / each;
      }
      if (a.count == 0 || (a.count < RO_MOST && i + 1 < count)) continue;
      for (int j = a.count; j < RO_MOST; ++j) a.first[j] = ~0u;
      if (across)
        hipLaunchKernelGGL(reorder_rows<true>, dim3((unsigned)groups), dim3(RO_NT), 0, stream, a);
      else
        hipLaunchKernelGGL(reorder_rows<false>, dim3((unsigned)groups), dim3(RO_NT), 0, stream, a);
      if (hipGetLastError() != hipSuccess) return MG_ERR_LAUNCH;
      a.count = 0, groups = 0;
    }
  }
  return MG_OK;
}

}  // extern "C"
