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
// 64 x 8 rows of 50257 in bf16, a fifth of them not read: 18 us for 41 MB and 6 for the selection.
// Of a wave's 12 us 1.5 are its first load, 1 the first bar's sort, 7 six tiles (a tile's exponentials
// and comparisons keep the vector units busy most of 1.1), 2 one or two sorts of what reached the bar.
//
// reorder_states: rows of up to 32 tensors a launch, in vectors of 16 bytes of the output, whose rows
// follow one another.  A vector lies in one row, read from wherever that starts, or holds the end of
// one and the start of the next, read byte by byte; rows of fewer bytes go in the largest units
// that sizes, strides and pointers allow.
#include "mg_paged.h"

namespace {

typedef u32x4 u32x4_any __attribute__((aligned(1)));

// ---- sorted lists over a wave -----------------------------------------------------------
__device__ __forceinline__ int bs_lane() { return threadIdx.x & (MG_WAVE - 1); }

// Lanes of `who` before this one.
__device__ __forceinline__ int bs_before(unsigned long long who) {
  return (int)__builtin_amdgcn_mbcnt_hi((unsigned)(who >> 32),
                                        __builtin_amdgcn_mbcnt_lo((unsigned)who, 0));
}

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
  Divisor by_lists, by_parts;     // K parts and parts
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
  // Vectors start at the row's first element, wherever that lies: who adds which elements, in which
  // order, then goes by their places in the row alone, so that equal rows have equal sums and their
  // candidates tie.  The last vector ends with the row; what it shares with the one before is that one's.
  // (By subtraction: of an integer, the compiler would not know that it points to global memory,
  // and its loads would be waited for wherever LDS is.)
  const int last = a.V < N ? 0 : a.V - N;
  // A row of less than a vector is read by elements; loads stay in the 16-byte line of its first.
  const T* const vectors = a.V < N ? x - (int)(((uintptr_t)x & 15) / sizeof(T)) : x;
  const int begin = part * a.per, stop = a.V - begin < a.per ? a.V : begin + a.per;

  Best<Key32> list;
  list.start(a.W);
  // No maximum is below the lowest number, so that a lane of -inf alone, or without an element,
  // has a sum of 0.
  float top = -3.402823466e38f, sum = 0.f;
  // A tile ahead; the first is on its way before it is known whether the row counts.
  u32x4 raw[VECTORS];
  auto load = [&](int at) {
#pragma unroll
    for (int i = 0; i < VECTORS; ++i) {
      const int e = at + (i * MG_WAVE + lane) * N;
      raw[i] = *(const u32x4_any*)(vectors + (e < last ? e : last));
    }
  };
  int kept = 0;
  if (begin < stop) load(begin);
  const float score = a.scores[b * a.ss[0] + k * a.ss[1]];
  if (bs_finished(a, b, k) || !bs_finite(score)) return;
  for (int at = begin; at < stop; at += TILE) {
    float v[ALL];
    float peak = -__builtin_inff();
    const bool whole = at + TILE <= stop;
#pragma unroll
    for (int i = 0; i < VECTORS; ++i) {
      const T* p = (const T*)&raw[i];
#pragma unroll
      for (int j = 0; j < N; ++j) v[i * N + j] = pg_float(p[j]);
    }
    load(at + TILE < stop ? at + TILE : begin);
    unsigned there = ~0u;
    if (!whole) {  // what is not in the row, or is there twice, adds nothing
      if (a.V < N) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = pg_float(x[j < a.V ? j : 0]);
      }
#pragma unroll
      for (int i = 0; i < ALL; ++i) {
        const int from = at + ((i / N) * MG_WAVE + lane) * N;
        const int e = (from < last ? from : last) + i % N;
        if (e >= from && e < stop) continue;
        v[i] = -__builtin_inff(), there &= ~(1u << i);
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
    bits &= there;
    for (unsigned long long who; (who = __ballot(bits != 0)) != 0; bits &= bits - 1) {
      const int i = __ffs(bits) - 1, to = hits + bs_before(who);
      const int from = at + (i / N * MG_WAVE + lane) * N;
      if (bits != 0 && to < BS_HITS) s_place[wave][to] = (from < last ? from : last) + i % N;
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
      const bool in = from ? i < ready : e < stop;
      const float value = pg_float(x[in ? e : 0]);
      list.offer(Key32{in ? ~(unsigned)e : 0u, in ? bs_order(value) : 0u});
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

// The candidates lie by their ranks in their lists (a part's), all lists' first ones ahead.  A first
// pass counts them by steps of how far they lie below the best score that a beam can give, and ends
// where all lists have fallen behind the steps that hold the W best; a second one puts those within
// reach, W and few more, into LDS, where each one's place is the number of those above it.  No chain
// is long: sorted lists over the waves' lanes, as for the rows, took 15 us of 31 for 16 searches of 16
// beams of 32771, 32 wide, where this takes 10 of 24; one search of 256 beams of 50257, 64 wide, took
// 151 us with both launches in place of 63.
// Eight waves and two candidates a thread: sixteen and four take 0.3 us less for the former,
// but 13.1 in place of 10.8 for 4 beams of 50257, 4 wide.
constexpr int BP_NW = 8, BP_NT = BP_NW * MG_WAVE, BP_HELD = 2, BP_CHUNK = BP_HELD * BP_NT;
constexpr int BP_STEPS = 256;
constexpr int BP_MOST = 256;  // keys in LDS before others come

// The candidates that may be among the W best, and how many of them are above each.
struct Pool {
  static constexpr int ROOM = BP_MOST + BP_NT;
  unsigned long long value[ROOM];
  unsigned index[ROOM];
  int rank[ROOM];
  int steps[BP_STEPS];
  int count, reach;
  int few;    // no more than BP_MOST are within reach
  int fresh;  // the last chunk, from 1, that has had some
  Key64 bar;  // the W-th of all before, once there have been more

  __device__ __forceinline__ Key64 at(int i) const {
    return Key64{index[i], (unsigned)value[i], (unsigned)(value[i] >> 32)};
  }
  __device__ __forceinline__ void put(int i, Key64 x) {
    value[i] = x.value(), index[i] = x.index, rank[i] = 0;
  }
  // All threads.  A wave takes 64 keys and those that it compares them with: all, or where there
  // are fewer keys than threads a part.
  __device__ __forceinline__ void order(int n) {
    const int wave = (int)mg_uniform(threadIdx.x / MG_WAVE);
    const int blocks = (n + MG_WAVE - 1) / MG_WAVE, cuts = blocks < BP_NW ? BP_NW / blocks : 1;
    const int each = (n + cuts - 1) / cuts;
    for (int u = wave; u < blocks * cuts; u += BP_NW) {
      const int cut = u / blocks, i = (u - cut * blocks) * MG_WAVE + bs_lane();
      const int end = (cut + 1) * each < n ? (cut + 1) * each : n;
      const Key64 x = at(i < n ? i : 0);
      int above = 0;
#pragma unroll 4
      for (int j = cut * each; j < end; ++j) above += at(j).above(x) ? 1 : 0;
      if (i < n) atomicAdd(&rank[i], above);
    }
    __syncthreads();
  }
};

__global__ __launch_bounds__(BP_NT) void beam_pick(BsArgs a) {
  constexpr int EACH = BP_STEPS / MG_WAVE;
  __shared__ Pool pool;
  enum { LIVE = 0, FINISHED = 1, DEAD = 2 };
  struct alignas(8) Beam {
    double score, log;  // log of the sum over exp(x - top)
    float top;
    int kind;
  };
  __shared__ Beam s_beam[BS_MAX_K];
  const int lane = bs_lane(), me = threadIdx.x;
  const int64_t b = blockIdx.x;
  const int lists = a.K * a.parts, all = lists * a.W;
  const unsigned long long* const keys = a.keys + b * all;
  // On their way together with all else: what other parts of the chip have just written is far away.
  unsigned long long raw[BP_HELD];
  auto load = [&](int at) {
#pragma unroll
    for (int i = 0; i < BP_HELD; ++i) raw[i] = keys[at + i * BP_NT + me < all ? at + i * BP_NT + me : 0];
  };
  load(0);
  // Sixteen lanes a row.
  for (int k0 = 0; k0 < a.K; k0 += BP_NW * 4) {
    const int k = k0 + (int)threadIdx.x / 16, in = threadIdx.x & 15;
    const int at = k < a.K ? k : a.K - 1;
    const float score = a.scores[b * a.ss[0] + at * a.ss[1]];
    const float2* st = a.stats + (b * a.K + at) * a.parts;
    // On their way before it is known whether the first launch has written them.
    const float2 none = make_float2(-__builtin_inff(), 0.f);
    const float2 x = in < a.parts ? st[in] : none, y = in + 16 < a.parts ? st[in + 16] : none;
    const bool finite = bs_finite(score), over = bs_finished(a, b, at);
    float m = fmaxf(x.x, y.x);
    double sum = 0.0;
    if (finite && !over) {
      for (int i = in + 32; i < a.parts; i += 16) m = fmaxf(m, st[i].x);
      m = fmaxf(m, mg_row_ror<8>(m));
      m = fmaxf(m, mg_row_ror<4>(m));
      m = fmaxf(m, mg_row_ror<2>(m));
      m = fmaxf(m, mg_row_ror<1>(m));
      sum = (double)x.y * (double)bs_exp(x.x - m) + (double)y.y * (double)bs_exp(y.x - m);
      for (int i = in + 32; i < a.parts; i += 16) sum += (double)st[i].y * (double)bs_exp(st[i].x - m);
      sum = bs_row_sum(sum);
    }
    if (in == 0 && k < a.K) {
      const double part = log(sum);
      const bool live = bs_finite(m) && fabs(part) < __builtin_inf();
      s_beam[k] = Beam{score, part, m, !finite ? DEAD : (over ? FINISHED : (live ? LIVE : DEAD))};
    }
  }
  for (int i = me; i < BP_STEPS; i += BP_NT) pool.steps[i] = 0;
  if (me == 0) pool.count = pool.fresh = pool.few = 0, pool.reach = BP_STEPS - 1, pool.bar = Key64{};
  __syncthreads();
  double most = -__builtin_inf();
  for (int k = lane; k < a.K; k += MG_WAVE) {
    const Beam beam = s_beam[k];
    if (beam.kind != DEAD) most = fmax(most, beam.kind == LIVE ? beam.score - beam.log : beam.score);
  }
#pragma unroll
  for (int d = 1; d < MG_WAVE; d *= 2) most = fmax(most, __shfl_xor(most, d));
  auto key = [&](double score, unsigned index) {
    const unsigned long long o = bs_order(score);
    return Key64{~index, (unsigned)o, (unsigned)(o >> 32)};
  };
  auto candidate = [&](int n, unsigned long long from) {
    const int r = (int)pg_div((unsigned)n, a.by_lists), at = n - r * lists;
    const int k = (int)pg_div((unsigned)at, a.by_parts);
    const Beam beam = s_beam[k];
    const bool live = beam.kind == LIVE, over = beam.kind == FINISHED;
    // In place of the parts of a beam that is not: its end, and the first tokens at -inf.
    const int token = over ? (r == 0 ? a.end : r - (r <= a.end ? 1 : 0)) : r;
    const bool there = live ? from != 0 : at == k * a.parts && token < a.V;
    // The difference first: a large top would swallow the logarithm.
    const double value = (double)bs_value((unsigned)(from >> 32)) - (double)beam.top - beam.log;
    const Key64 x = key(live || (over && r == 0) ? beam.score + (live ? value : 0.0) : -__builtin_inf(),
                        (unsigned)k * (unsigned)a.V + (live ? ~(unsigned)from : (unsigned)token));
    return x.pick(there, Key64{});
  };
  // How far below the beams' best scores a candidate lies, in steps of an eighth of an octave from
  // 2^-8 on: the W best are in the first steps that hold W, and those hold few more.
  auto step = [&](Key64 x) {
    const float d = (float)(most - bs_value(x.value()));
    const int s = (int)(__float_as_uint(d) >> 20) - ((127 - 8) << 3);
    return d < 0.00390625f ? 0 : (s < BP_STEPS ? s : BP_STEPS - 1);
  };
  Key64 held[BP_HELD];
  auto value_all = [&](int at) {
#pragma unroll
    for (int i = 0; i < BP_HELD; ++i) {
      const int n = at + i * BP_NT + me;
      held[i] = candidate(n < all ? n : 0, raw[i]);
      held[i] = held[i].pick(n < all, Key64{});
    }
  };
  int end = 0, reach = BP_STEPS - 1;
  bool few = false;
  for (int at = 0; at < all; at += BP_CHUNK) {
    if (at) load(at);
    value_all(at);
    bool fresh = false;
#pragma unroll
    for (int i = 0; i < BP_HELD; ++i) {
      const int s = step(held[i]);
      if (held[i].index == 0 || s >= BP_STEPS - 1 || s > reach) continue;
      atomicAdd(&pool.steps[s], 1);
      fresh = true;
    }
    if (fresh) pool.fresh = at + 1;
    __syncthreads();
    // Nothing new within reach among as many candidates as there are lists: some rank of every list,
    // so that none behind it is.
    if (reach < BP_STEPS - 1 && pool.fresh != at + 1) {
      if (at + BP_CHUNK - end >= lists) break;
      continue;
    }
    end = at + BP_CHUNK;
    if (me < MG_WAVE) {
      int n[EACH], sum = 0;
#pragma unroll
      for (int i = 0; i < EACH; ++i) sum += n[i] = pool.steps[me * EACH + i];
      int before = sum;
#pragma unroll
      for (int d = 1; d < MG_WAVE; d *= 2) {
        const int o = __shfl_up(before, d);
        before += lane >= d ? o : 0;
      }
      // The step at which W are reached; the last one, whose are not counted, if none is.
      const unsigned long long who = __ballot(before >= a.W);
      if (who && me == __ffsll(who) - 1) {
        before -= sum;
        int s = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          const bool on = before < a.W;
          before += on ? n[i] : 0, s += on ? 1 : 0;
        }
        pool.reach = me * EACH + s - 1, pool.few = before <= BP_MOST;
      }
    }
    __syncthreads();
    reach = pool.reach, few = pool.few != 0;
  }
  end = end < all ? end : all;
#pragma unroll 1
  for (int at = 0;; at += BP_NT) {
    const int i = at / BP_NT % BP_HELD;
    if (i == 0 && all > BP_CHUNK) load(at), value_all(at);
    Key64 one = held[0];
#pragma unroll
    for (int j = 1; j < BP_HELD; ++j) one = held[j].pick(i == j, one);
    const bool in = one.above(pool.bar) && step(one) <= reach;
    const unsigned long long who = __ballot(in);
    if (who) {
      int to = 0;
      if (lane == 0) to = atomicAdd(&pool.count, __popcll(who));
      to = (int)bs_read((unsigned)to, 0) + bs_before(who);
      if (in) pool.put(to, one);
    }
    const bool more = at + BP_NT < end;
    if (more && few) continue;
    __syncthreads();
    const int n = pool.count;
    if (more && n <= BP_MOST) {
      __syncthreads();
      continue;
    }
    pool.order(n);
    Key64 x[Pool::ROOM / BP_NT + 1];
    int rank[Pool::ROOM / BP_NT + 1];
#pragma unroll
    for (int i = 0; i <= Pool::ROOM / BP_NT; ++i) {
      const int from = me + i * BP_NT;
      rank[i] = from < n ? pool.rank[from] : a.W;
      x[i] = pool.at(from < n ? from : 0);
    }
    if (!more) {
#pragma unroll
      for (int i = 0; i <= Pool::ROOM / BP_NT; ++i) {
        if (rank[i] >= a.W) continue;
        const unsigned flat = ~x[i].index;
        const int k = (int)(flat / (unsigned)a.V), token = (int)(flat - (unsigned)k * (unsigned)a.V);
        const int64_t to = b * a.W + rank[i];
        a.out[to] = (float)bs_value(x[i].value());
        a.parents[to] = k, a.tokens[to] = token;
        if (a.done) a.done[to] = token == a.end || bs_finished(a, b, k);
      }
      return;
    }
    // The W best go on, and the last of them is the bar.
    __syncthreads();
#pragma unroll
    for (int i = 0; i <= Pool::ROOM / BP_NT; ++i) {
      if (rank[i] >= a.W) continue;
      pool.put(rank[i], x[i]);
      if (rank[i] == a.W - 1) pool.bar = x[i];
    }
    if (me == 0) pool.count = a.W;
    __syncthreads();
  }
}

// Waves of a row: two for each of the chip's 1024 vector units over all rows, none with less than
// a tile.  (64 x 8 rows of 50257 in bf16, both launches in a graph: 23.4 us; four for each 24.4, one
// 25.5.  16 x 16 of 32771 in fp32, 32 wide: 24.2, four, with more first tiles and candidates, 25.2, one
// 24.8.)
int bs_parts(int64_t rows, int V, int tile) {
  const int64_t want = (2048 + rows - 1) / rows;
  const int64_t most = ((int64_t)V + tile - 1) / tile;
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
  const int64_t per = (V + a.parts - 1) / a.parts;
  a.per = (int)((per + tile - 1) / tile * tile);
  a.parts = (int)((V + a.per - 1) / a.per);
  a.by_lists = pg_divisor(K * a.parts), a.by_parts = pg_divisor(a.parts);
  a.keys = (unsigned long long*)ws;
  a.stats = (float2*)(a.keys + B * K * a.parts * W);
  a.out = out, a.parents = parents, a.tokens = tokens, a.done = (unsigned char*)done;
  const dim3 grid((unsigned)((B * K * a.parts + BS_NW - 1) / BS_NW)), nt(BS_NT);
  if (dtype == 0) hipLaunchKernelGGL(beam_rows<float>, grid, nt, 0, stream, a);
  else if (dtype == 1) hipLaunchKernelGGL(beam_rows<Bf16>, grid, nt, 0, stream, a);
  else hipLaunchKernelGGL(beam_rows<Fp16>, grid, nt, 0, stream, a);
  if (hipGetLastError() != hipSuccess) return MG_ERR_LAUNCH;
  hipLaunchKernelGGL(beam_pick, dim3((unsigned)B), dim3(BP_NT), 0, stream, a);
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
