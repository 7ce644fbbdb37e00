// Attention of each sequence's newest token over a paged cache (gfx950).
//
//   s_j = scale q . k_j;  o = sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s)
// over a sequence's last tokens, for each head; the heads of a group share a key head.
//
// Bound by memory: every key and value is read once (by each 16 queries of a larger group).  The unit of
// work is a tile of 32 tokens (16 in fp32) of one key head, held by one wave, for 16 query heads of the
// group on the matrix cores: rows beyond the group are idle there, but at 16 rows a bf16 tile of 16 KB
// costs a SIMD some 350 cycles of matrix instructions, where its share of the memory's rate is 7000.
//
// Sums as the matrix cores take them (lane = 16 g + c, g < 4):
// * A lane loads its tile's tokens 4 g + j (and 16 + 4 g + j), 1/16 of a row (chunk c) of each, so
//   that a wave's load covers whole rows of four tokens.
// * S^T = K Q^T.  The keys go through LDS, rows padded by 16 bytes, private to the wave: no
//   barrier.  The result has query c in lane's column c, tokens 4 g + i in its registers.
// * O^T = V^T P^T.  The tokens that a lane's probabilities belong to are the tokens whose values
//   it loaded, so neither moves between lanes: the product's rows are the elements E c + e of
//   all chunks c at one e (E elements a chunk), a fragment of them is a lane's element e of
//   each of its tokens.
// * Half types' probabilities are summands of their type, three in bf16 and two in fp16, so that the
//   rounding is 2^-24 or 2^-22 of them: one's is as large as the result's own, and two in bf16 (2^-16)
//   show where values cancel.  (524287 tokens of 8 key heads in bf16: 368 us, with two 366.)  In fp16,
//   which has nothing below 2^-24, they and their sum are 2^15 times as large: weights down to 2^-40 of
//   the largest count in the products as they do in the sum.
// Maxima, sums and O are fp32, with O scaled again only where a maximum rises.
//
// Work is divided on the device, where the lengths are: the steps (four tiles, one for each wave
// of a workgroup) of all sequences and key heads form one row, cut into equal shares for as
// many workgroups as the chip holds at once.  So ragged batches, one long sequence and many short
// ones all keep every CU busy, and the host looks at no length.  A share that holds all steps of
// a head writes its output; others leave (max, sum, O) to a second launch, in a fixed order.
// A share's loads run on over the ends of its pieces: the next step's keys and values, and the pages
// of the one after it, are on their way whichever piece they are of.
//
// bf16, heads of 128, 4 queries a key head: 64 sequences of up to 8192 tokens (501 MB) 97 to 104 us, 5 TB/s,
// and 5 for the join; 524287 tokens of 8 key heads, 2 queries each (2.1 GB), 358 to 370 us, 5.9 TB/s.  A
// copy reaches 5.13.
#include "mg_paged.h"

namespace {

constexpr int PA_NW = 4, PA_NT = PA_NW * MG_WAVE, PA_ROWS = 16;

struct PaArgs {
  const void *q, *k, *v;
  void* o;
  Ints pages, lengths;
  int64_t qs[2];          // strides in elements: sequence, head
  int64_t ks[3], vs[3];   // page, head, slot
  int64_t page_stride;
  int64_t B, N;
  int64_t room;           // tokens that a row of pages holds
  int64_t window;         // 0: all tokens
  Divisor P;
  int H, Hk, group, tiles_q, dk, dv;
  float scale;            // times log2 e
  int shares;
  float* part;            // (2 shares, rows, dv) sums, then (2 shares, rows, 2) maxima and sums
  int rows;
  int few_steps;          // whether the sequences' steps cannot pass 2^31
};

// ---- element types ---------------------------------------------------------------------
template <typename T>
struct Elem;
template <>
struct Elem<Bf16> {
  static constexpr int KEYS = 32, PAD = 8;
  static constexpr float WEIGHT = 1.f;
  static constexpr int PLANES = 3;
  typedef bf16x8 Frag;
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float low(unsigned u) { return __uint_as_float(u << 16); }
  static __device__ __forceinline__ float high(unsigned u) { return __uint_as_float(u & 0xffff0000u); }
};
template <>
struct Elem<Fp16> {
  static constexpr int KEYS = 32, PAD = 8;
  static constexpr float WEIGHT = 32768.f;  // of a score that is the maximum
  static constexpr int PLANES = 2;
  typedef f16x8 Frag;
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float low(unsigned u) {
    return (float)__builtin_bit_cast(f16x2, u)[0];
  }
  static __device__ __forceinline__ float high(unsigned u) {
    return (float)__builtin_bit_cast(f16x2, u)[1];
  }
};
template <>
struct Elem<float> {
  static constexpr int KEYS = 16, PAD = 4;
  static constexpr float WEIGHT = 1.f;
};

// A lane's chunk of a row: E elements in registers of 32 bits.
template <typename T, int E>
struct Chunk {
  static constexpr int W = E * sizeof(T) / 4;
  unsigned w[W];
};

// Chunk c of a row of d elements.  VEC: d, strides and pointers are multiples of 16 bytes (8
// where a chunk is 8), so that a vector lies in the row or behind it as a whole.  What lies
// behind is read from the row's start and set to 0 later (pa_clear).
template <typename T, int E, bool VEC>
__device__ __forceinline__ void pa_load(const T* row, int c, int d, Chunk<T, E>& x) {
  constexpr int W = Chunk<T, E>::W;
  if constexpr (VEC) {
    constexpr int L = W < 4 ? W : 4, VE = L * 4 / sizeof(T);
#pragma unroll
    for (int i = 0; i < W / L; ++i) {
      const int at = c * E + i * VE;
      const T* p = row + (at < d ? at : 0);
      if constexpr (L == 2) {
        const u32x2 v = *(const u32x2*)p;
        x.w[0] = v[0], x.w[1] = v[1];
      } else {
        const u32x4 v = *(const u32x4*)p;
#pragma unroll
        for (int j = 0; j < 4; ++j) x.w[4 * i + j] = v[j];
      }
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int at = c * E + i;
      x.w[i] = ((const unsigned*)row)[at < d ? at : 0];
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int at = c * E + 2 * i;
      const unsigned lo = ((const u16*)row)[at < d ? at : 0];
      const unsigned hi = ((const u16*)row)[at + 1 < d ? at + 1 : 0];
      x.w[i] = lo | hi << 16;
    }
  }
}
// Elements from d on become 0.
template <typename T, int E>
__device__ __forceinline__ void pa_clear(int c, int d, Chunk<T, E>& x) {
#pragma unroll
  for (int i = 0; i < Chunk<T, E>::W; ++i) {
    if constexpr (sizeof(T) == 4) {
      x.w[i] = c * E + i < d ? x.w[i] : 0u;
    } else {
      const int at = c * E + 2 * i;
      x.w[i] = at + 1 < d ? x.w[i] : (at < d ? x.w[i] & 0xffffu : 0u);
    }
  }
}

__device__ __forceinline__ float pa_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// Maximum and sum over the lanes of one column (g of lane = 16 g + c), in all of them.
__device__ __forceinline__ float pa_max(float x) {
  unsigned u = __float_as_uint(x);
  auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  u = __float_as_uint(x);
  r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pa_wave_max(float x) {
  x = fmaxf(x, mg_row_ror<8>(x));
  x = fmaxf(x, mg_row_ror<4>(x));
  x = fmaxf(x, mg_row_ror<2>(x));
  return pa_max(fmaxf(x, mg_row_ror<1>(x)));
}
__device__ __forceinline__ float pa_sum(float x) { return mg_pair_sum<32>(mg_pair_sum<16>(x)); }

// ---- the division of work --------------------------------------------------------------
// Values that every lane holds, in scalar registers.
__device__ __forceinline__ int64_t pa_uniform(int64_t x) {
  return (int64_t)((uint64_t)mg_uniform((unsigned)((uint64_t)x >> 32)) << 32 | mg_uniform((unsigned)x));
}

// A sequence's tokens that count, [first, end), and the steps of SPAN tokens that hold them.
struct PaSeq {
  int first, end;
  int step0, steps;  // of one key head
  int bad;           // longer than its pages
};
template <int SPAN>
__device__ __forceinline__ PaSeq pa_seq(const PaArgs& a, int64_t b) {
  PaSeq s;
  const int64_t n = a.lengths[b];
  s.bad = n > a.room;
  s.end = (int)(n < 0 ? 0 : (n > a.room ? a.room : n));
  s.first = a.window && s.end > a.window ? s.end - (int)a.window : 0;
  s.step0 = (unsigned)s.first / SPAN;
  s.steps = s.end > 0 ? (int)((unsigned)(s.end + SPAN - 1) / SPAN) - s.step0 : 0;
  return s;
}
template <int SPAN>
__device__ __forceinline__ PaSeq pa_seq_uniform(const PaArgs& a, int64_t b) {
  const PaSeq s = pa_seq<SPAN>(a, b);
  return PaSeq{(int)mg_uniform(s.first), (int)mg_uniform(s.end), (int)mg_uniform(s.step0),
               (int)mg_uniform(s.steps), (int)mg_uniform(s.bad)};
}

// The steps of sequences [b0, b0 + n), the lanes taking runs of `run` of them, summed over the
// lanes up to each, itself included.  (No LDS, no barrier: each wave looks for itself.)
template <int SPAN>
__device__ __forceinline__ int64_t pa_steps(const PaArgs& a, int64_t b0, int64_t n, int64_t run) {
  const int lane = threadIdx.x & (MG_WAVE - 1);
  int64_t sum = 0;
  for (int64_t i = lane * run; i < (lane + 1) * run && i < n; ++i) sum += pa_seq<SPAN>(a, b0 + i).steps;
  if (a.few_steps) {  // 32 bits hold them all
    int x = (int)sum;
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    const int t0 = __builtin_amdgcn_readlane(x, 15), t1 = __builtin_amdgcn_readlane(x, 31);
    const int t2 = __builtin_amdgcn_readlane(x, 47), row = lane >> 4;
    return x + (row > 0 ? t0 : 0) + (row > 1 ? t1 : 0) + (row > 2 ? t2 : 0);
  }
#pragma unroll
  for (int d = 1; d < MG_WAVE; d *= 2) {
    const int64_t up = __shfl_up(sum, d);
    sum += lane >= d ? up : 0;
  }
  return sum;
}
__device__ __forceinline__ int64_t pa_lane(int64_t x, int lane) {  // the same lane for all
  return (int64_t)((uint64_t)(unsigned)__builtin_amdgcn_readlane((int)((uint64_t)x >> 32), lane) << 32 |
                   (unsigned)__builtin_amdgcn_readlane((int)x, lane));
}
// All sequences' steps as one row, a sequence's pairs of a key head and 16 of its queries one
// after another.  The sequence that holds step `at`, and its first step.
struct PaPlace {
  int64_t b, before;
};
template <int SPAN>
__device__ __forceinline__ int64_t pa_all(const PaArgs& a, int64_t pairs, int64_t& sums, int64_t& run) {
  run = (a.B + MG_WAVE - 1) / MG_WAVE;
  sums = pa_steps<SPAN>(a, 0, a.B, run);
  return pa_lane(sums, MG_WAVE - 1) * pairs;
}
template <int SPAN>
__device__ __forceinline__ PaPlace pa_find(const PaArgs& a, int64_t pairs, int64_t sums, int64_t run,
                                           int64_t at) {
  PaPlace p = {0, 0};
  int64_t n = a.B;
  for (;;) {
    // The run that holds it: the lanes before have all theirs before it.
    const int lane = __popcll(__ballot(p.before + sums * pairs <= at));
    if (lane > 0) p.before += pa_lane(sums, lane - 1) * pairs;
    p.b += lane * run;
    if (run == 1) return p;
    n = n - lane * run < run ? n - lane * run : run;
    run = (run + MG_WAVE - 1) / MG_WAVE;
    sums = pa_steps<SPAN>(a, p.b, n, run);
  }
}

// A step of a sequence's: its pair, and which of that.
struct PaPair {
  int pair, step;
};
__device__ __forceinline__ PaPair pa_pair(int64_t in, int steps) {
  in = pa_uniform(in);
  const int pair = in >> 32 ? (int)(in / steps) : (int)((unsigned)in / (unsigned)steps);
  return PaPair{pair, (int)(in - (int64_t)pair * steps)};
}

// Share w of n holds the steps [w all / n, (w + 1) all / n); no share is empty, as n <= all.
__device__ __forceinline__ int pa_shares_used(const PaArgs& a, int64_t all) {
  return all < a.shares ? (int)all : a.shares;
}
// Quotients of 32 bits where they suffice: those of 64 take some 100 instructions.
__device__ __forceinline__ int64_t pa_share(int64_t w, int64_t all, int n) {
  const uint64_t x = (uint64_t)w * (uint64_t)all;
  return x >> 32 ? (int64_t)(x / (unsigned)n) : (int64_t)((unsigned)x / (unsigned)n);
}
__device__ __forceinline__ int pa_holder(int64_t step, int64_t all, int n) {
  const uint64_t x = (uint64_t)(step + 1) * (unsigned)n - 1;
  return (x | (uint64_t)all) >> 32 ? (int)(x / (uint64_t)all) : (int)((unsigned)x / (unsigned)all);
}

// ---- the main kernel -------------------------------------------------------------------
// Workgroups that a CU holds: at 256 a step, its successor, queries and outputs take 300 registers.
constexpr int pa_groups(int dk, int dv) { return dv > 128 ? 1 : (dk > 64 ? 2 : 3); }
template <typename T, int DK, int DV>
struct PaShape {
  static constexpr int KEYS = Elem<T>::KEYS;      // tokens of a tile
  static constexpr int SPAN = KEYS * PA_NW;       // of a step
  static constexpr int EK = DK / 16, EV = DV / 16;  // elements of a chunk
  static constexpr int NK = KEYS / 4;             // tokens of a lane
  static constexpr int LD = DK + Elem<T>::PAD;    // elements of a key's row in LDS
  static constexpr int OLD = DV + 4;              // floats of an output row in LDS
  static constexpr int BYTES = KEYS * LD * sizeof(T);  // of a wave
  // Workgroups of a CU.
  static constexpr int GROUPS = pa_groups(DK, DV);
  static_assert(DV <= DK && PA_ROWS * OLD * 4 <= BYTES, "the outputs lie where the keys were");
};

// One step of a share, of a piece of one pair's steps: uniform values.
struct PaStep {
  PaSeq seq;
  int64_t b, left;       // sequence; steps of the share behind this piece
  int hk, tile_q;        // the pair
  int here, todo;        // steps of the piece, and those from this one on
  int base;              // this wave's first token
  bool valid;
};

// FOURS: pages hold a multiple of 4 tokens, so that a lane's tokens 4 g + j share one.
template <typename T, int DK, int DV, bool VEC, bool FOURS>
__global__ __launch_bounds__(PA_NT, (PaShape<T, DK, DV>::GROUPS)) void paged_attention(PaArgs a) {
  typedef PaShape<T, DK, DV> S;
  constexpr int KEYS = S::KEYS, EK = S::EK, EV = S::EV, NK = S::NK, LD = S::LD, OLD = S::OLD;
  constexpr int SPAN = S::SPAN;
  constexpr int NG = NK / 4;               // groups of four tokens of a lane
  constexpr int NP = FOURS ? NG : NK;      // pages of a lane
  constexpr int QW = DK * sizeof(T) / 64;  // vectors of 16 bytes of a query's fragment
  typedef Chunk<T, EK> CK;
  typedef Chunk<T, EV> CV;
  __shared__ alignas(16) unsigned char s_tile[PA_NW][S::BYTES];
  __shared__ float s_max[PA_NW][PA_ROWS], s_sum[PA_NW][PA_ROWS];

  const int lane = threadIdx.x & (MG_WAVE - 1), wave = (int)mg_uniform(threadIdx.x / MG_WAVE);
  const int c = lane & 15, g = lane >> 4;
  T* const tile = (T*)s_tile[wave];
  float* const sums = (float*)s_tile[wave];
  const bool short_k = DK != a.dk;

  // The outputs of sequences without a token.
  for (int64_t b0 = blockIdx.x; b0 < a.B; b0 += (int64_t)gridDim.x * PA_NT) {
    const int64_t b = b0 + (int64_t)gridDim.x * threadIdx.x;
    unsigned long long empty = __ballot(b < a.B && a.lengths[b < a.B ? b : b0] <= 0);
    for (; empty != 0; empty &= empty - 1) {
      const int64_t at = b0 + (int64_t)gridDim.x * (wave * MG_WAVE + __ffsll(empty) - 1);
      const int64_t n = a.H * (int64_t)a.dv;
      T* const dst = (T*)a.o + at * n;
      for (int64_t x = lane; x < n; x += MG_WAVE) dst[x] = pg_round<T>(0.f);
    }
  }

  // This share's first step.
  PaStep now;
  {
    const int64_t pairs = (int64_t)a.Hk * a.tiles_q;
    int64_t steps, run;
    const int64_t all = pa_all<SPAN>(a, pairs, steps, run);
    const int shares = pa_shares_used(a, all);
    if ((int)blockIdx.x >= shares) return;
    const int64_t at = pa_share(blockIdx.x, all, shares);
    now.left = pa_share(blockIdx.x + 1, all, shares) - at;
    const PaPlace p = pa_find<SPAN>(a, pairs, steps, run, at);
    now.b = pa_uniform(p.b);
    now.seq = pa_seq_uniform<SPAN>(a, now.b);
    const PaPair pair = pa_pair(at - p.before, now.seq.steps);
    now.hk = pair.pair / a.tiles_q, now.tile_q = pair.pair - now.hk * a.tiles_q;
    now.todo = pair.step;  // for now
    now.valid = true;
  }
  auto open = [&](PaStep& s, int step) {  // a piece from that step of its pair on
    const int n = s.seq.steps - step;
    s.here = s.left < n ? (int)s.left : n, s.todo = s.here, s.left -= s.here;
    s.base = (s.seq.step0 + step) * SPAN + wave * KEYS;
  };
  auto advance = [&](PaStep& s) {
    if (--s.todo > 0) {
      s.base += SPAN;
    } else if (s.left > 0) {
      if (++s.tile_q == a.tiles_q) s.tile_q = 0, ++s.hk;
      if (s.hk == a.Hk) {
        s.hk = 0;
        do s.seq = pa_seq_uniform<SPAN>(a, ++s.b);
        while (s.seq.steps == 0);
      }
      open(s, 0);
    } else {
      s.valid = false, s.todo = 1, s.base = s.seq.end;  // every lane asks for the last token
    }
  };
  open(now, now.todo);
  PaStep next = now;
  advance(next);
  PaStep far = next;
  advance(far);

  CK kr[NK];
  CV vr[NK];
  unsigned page[NP], upper[NP];
  int64_t vo[NP];
  unsigned bad = 0, bad_next = 0;  // tokens of this lane whose page is not in the cache
  u32x4 qf[QW];
  auto token = [&](const PaStep& s, int i) {  // behind the last token, one of its page
    const int key = s.base + (FOURS ? 16 * i + 4 * g : 16 * (i / 4) + 4 * g + i % 4);
    return key < s.seq.end ? key : (FOURS ? (s.seq.end - 1) & ~3 : s.seq.end - 1);
  };
  // The pages of a step's tokens: both words without a branch, where the loads would be waited
  // for.  The upper one of an int64 that is a page is 0, as N < 2^31; of an int32 the same word
  // stands for it.
  auto look = [&](const PaStep& s) {
    const unsigned* const row = (const unsigned*)a.pages.p + ((s.b * a.page_stride) << a.pages.wide);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const unsigned* const p = row + ((size_t)pg_div((unsigned)token(s, i), a.P) << a.pages.wide);
      page[i] = p[0], upper[i] = p[a.pages.wide];
    }
  };
  // Loads of the keys, from the pages that were looked up; the values' places are kept.
  auto keys = [&](const PaStep& s) {
    const T* const kc = (const T*)a.k + s.hk * a.ks[1];
    bad_next = 0;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int key = token(s, i);
      const int slot = key - (int)(pg_div((unsigned)key, a.P) * a.P.d);
      const bool in = page[i] < (unsigned)a.N && (!a.pages.wide || upper[i] == 0);
      bad_next |= in ? 0u : 1u << i;
      const int64_t p = in ? page[i] : 0;
      vo[i] = s.hk * a.vs[1] + p * a.vs[0] + slot * a.vs[2];
      const T* row = kc + p * a.ks[0] + slot * a.ks[2];
      if constexpr (FOURS) {
#pragma unroll
        for (int j = 0; j < 4; ++j) pa_load<T, EK, VEC>(row + j * a.ks[2], c, a.dk, kr[4 * i + j]);
      } else {
        pa_load<T, EK, VEC>(row, c, a.dk, kr[i]);
      }
    }
  };
  auto values = [&] {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const T* row = (const T*)a.v + vo[i];
      if constexpr (FOURS) {
#pragma unroll
        for (int j = 0; j < 4; ++j) pa_load<T, EV, VEC>(row + j * a.vs[2], c, a.dv, vr[4 * i + j]);
      } else {
        pa_load<T, EV, VEC>(row, c, a.dv, vr[i]);
      }
    }
  };
  // Queries: column c, the elements that a key's fragment holds, 0 behind the head's.
  auto queries = [&](const PaStep& s) {
    const int q0 = s.hk * a.group + s.tile_q * PA_ROWS, rows = a.group - s.tile_q * PA_ROWS;
    const T* row = (const T*)a.q + s.b * a.qs[0] + (int64_t)(q0 + (c < rows ? c : 0)) * a.qs[1];
    constexpr int VE = 16 / sizeof(T);
    // Places in a row are formed anew for each piece: kept, they take a register an element.
    int chunk = g;
    asm volatile("" : "+v"(chunk));
#pragma unroll
    for (int s = 0; s < QW; ++s) {
      const int at = (4 * s + chunk) * VE;
      if constexpr (VEC && CK::W == 2) {  // a row is a multiple of 8 bytes
        const u32x2 x = *(const u32x2*)(row + (at < a.dk ? at : 0));
        const u32x2 y = *(const u32x2*)(row + (at + VE / 2 < a.dk ? at + VE / 2 : 0));
        const bool in = at < a.dk, all = at + VE / 2 < a.dk;
        qf[s] = u32x4{in ? x[0] : 0, in ? x[1] : 0, all ? y[0] : 0, all ? y[1] : 0};
      } else if constexpr (VEC) {
        const u32x4 x = *(const u32x4*)(row + (at < a.dk ? at : 0));
        qf[s] = at < a.dk ? x : u32x4{0, 0, 0, 0};
      } else {
        Chunk<T, VE> x;
        pa_load<T, VE, false>(row, 4 * s + chunk, a.dk, x);
        pa_clear<T, VE>(4 * s + chunk, a.dk, x);
        qf[s] = u32x4{x.w[0], x.w[1], x.w[2], x.w[3]};
      }
    }
  };

  look(now);
  queries(now);
  keys(now);
  values();
  look(next);
  f32x4 o[EV];
#pragma unroll
  for (int e = 0; e < EV; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
  float top = -__builtin_inff(), sum = 0.f;
  bool head = true;  // the share's first piece
  for (;;) {
    const int base = now.base, first = now.seq.first, end = now.seq.end;
    // Keys into LDS, and the next step's on their way, whichever piece it is of.
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      if (short_k) pa_clear<T, EK>(c, a.dk, kr[j]);
      T* dst = tile + (16 * (j / 4) + 4 * g + j % 4) * LD + c * EK;
      if constexpr (CK::W == 2) {
        *(u32x2*)dst = u32x2{kr[j].w[0], kr[j].w[1]};
      } else {
#pragma unroll
        for (int w = 0; w < CK::W; w += 4)
          *(u32x4*)((unsigned*)dst + w) =
              u32x4{kr[j].w[w], kr[j].w[w + 1], kr[j].w[w + 2], kr[j].w[w + 3]};
      }
    }
    bad = bad_next;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_sched_barrier(0);
    // Under no condition: loads under one would be waited for where the branches meet.
    keys(next);
    look(far);
    // A wave without a token here (the ends of the row of tokens) has nothing to add.
    if (base < end && base + KEYS > first) {
      f32x4 s[NG];
#pragma unroll
      for (int t = 0; t < NG; ++t) {
        s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < QW; ++x) {
          const u32x4 kf = *(const u32x4*)((const unsigned char*)(tile + (16 * t + c) * LD) + 64 * x + 16 * g);
          if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf[e]),
                                                          __uint_as_float(qf[x][e]), s[t], 0, 0, 0);
          } else {
            s[t] = Elem<T>::mma(kf, qf[x], s[t]);
          }
        }
      }
      float p[NK], peak = -__builtin_inff();
      const bool whole = base >= first && base + KEYS <= end && __ballot(bad != 0) == 0;
#pragma unroll
      for (int j = 0; j < NK; ++j) p[j] = s[j / 4][j % 4] * a.scale;
      if (!whole) {
#pragma unroll
        for (int j = 0; j < NK; ++j) {
          const int key = base + 16 * (j / 4) + 4 * g + j % 4;
          const bool live = key >= first && key < end;
          const bool lost = bad >> (FOURS ? j / 4 : j) & 1;
          p[j] = live ? (lost ? __builtin_nanf("") : p[j]) : -__builtin_inff();
          // 0 times a value that is not finite would be a NaN.
#pragma unroll
          for (int w = 0; w < CV::W; ++w) vr[j].w[w] = live ? vr[j].w[w] : 0u;
        }
      }
#pragma unroll
      for (int j = 0; j < NK; ++j) peak = fmaxf(peak, p[j]);
      peak = fmaxf(pa_max(peak), top);
      const float from = peak == -__builtin_inff() ? 0.f : peak;
      if (__ballot(peak > top) != 0) {
        const float down = pa_exp2(top - from);
        sum *= down;
#pragma unroll
        for (int e = 0; e < EV; ++e) o[e] *= down;
        top = peak;
      }
#pragma unroll
      for (int j = 0; j < NK; ++j) {
        p[j] = Elem<T>::WEIGHT * pa_exp2(p[j] - from);
        sum += p[j];
      }
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < NK; ++j)
#pragma unroll
          for (int e = 0; e < EV; ++e)
            o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[j].w[e]), p[j], o[e], 0,
                                                        0, 0);
      } else {
        u32x4 plane[Elem<T>::PLANES];
#pragma unroll
        for (int n = 0; n < Elem<T>::PLANES; ++n) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            plane[n][j] = pg_pack<T>(p[2 * j], p[2 * j + 1]);
            p[2 * j] -= Elem<T>::low(plane[n][j]), p[2 * j + 1] -= Elem<T>::high(plane[n][j]);
          }
        }
#pragma unroll
        for (int e = 0; e < EV; ++e) {
          u32x4 vf;
#pragma unroll
          for (int j = 0; j < 4; ++j)  // element e of tokens 2 j and 2 j + 1
            vf[j] = __builtin_amdgcn_perm(vr[2 * j + 1].w[e / 2], vr[2 * j].w[e / 2],
                                          e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int n = 0; n < Elem<T>::PLANES; ++n) o[e] = Elem<T>::mma(vf, plane[n], o[e]);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    values();
    __builtin_amdgcn_wave_barrier();
    if (now.todo == 1) {
      // The piece's end: the waves' sums meet in LDS, where the keys were.
      if (next.valid) queries(next);
      sum = pa_sum(sum);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int e = 0; e < EV; e += 4)
          *(f32x4*)(sums + c * OLD + EV * (4 * g + i) + e) =
              f32x4{o[e][i], o[e + 1][i], o[e + 2][i], o[e + 3][i]};
      }
      if (lane < PA_ROWS) s_max[wave][lane] = top, s_sum[wave][lane] = sum;
      __syncthreads();
      const bool done = now.here == now.seq.steps;
      const int q0 = now.tile_q * PA_ROWS, rows = a.group - q0 < PA_ROWS ? a.group - q0 : PA_ROWS;
      const int64_t slot = 2 * (int64_t)blockIdx.x + (head ? 0 : 1);
      for (int n = threadIdx.x; n < rows * (DV / 4); n += PA_NT) {
        const int r = n / (DV / 4), x = 4 * (n - r * (DV / 4));
        if (x >= a.dv) continue;
        float m = s_max[0][r];
#pragma unroll
        for (int w = 1; w < PA_NW; ++w) m = fmaxf(m, s_max[w][r]);
        const float from = m == -__builtin_inff() ? 0.f : m;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < PA_NW; ++w) {
          const float down = pa_exp2(s_max[w][r] - from);
          l += down * s_sum[w][r];
          v += down * *(const f32x4*)((const float*)s_tile[w] + r * OLD + x);
        }
        if (done) {
          T* dst = (T*)a.o + (now.b * a.H + now.hk * a.group + q0 + r) * (int64_t)a.dv;
          const float inv = now.seq.bad ? __builtin_nanf("") : 1.f / l;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (x + e < a.dv) dst[x + e] = pg_round<T>(v[e] * inv);
        } else {
          float* dst = a.part + (slot * a.rows + r) * a.dv;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (x + e < a.dv) dst[x + e] = v[e];
          if (x == 0) {
            float* stat = a.part + 2 * (int64_t)a.shares * a.rows * a.dv + (slot * a.rows + r) * 2;
            stat[0] = m, stat[1] = l;
          }
        }
      }
      if (!next.valid) return;
      __syncthreads();
      head = false;
      top = -__builtin_inff(), sum = 0.f;
#pragma unroll
      for (int e = 0; e < EV; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    now = next, next = far;
    if (far.valid) advance(far);
  }
}

// Joins the pieces of the pairs that are cut in two or more.  Where pairs are few and pieces many, a
// workgroup for each pair and query head (BY_PAIR, at most 64 sequences); else a wave for each start
// of a share, which cuts a pair or does not, and query head.  (A workgroup for each of all heads,
// most of which are whole, took 131 us for 1024 sequences of 256 tokens and 16 heads, where the
// main kernel takes 104 and this 6.)
template <typename T, int SPAN, bool BY_PAIR>
__global__ __launch_bounds__(PA_NT) void paged_attention_join(PaArgs a) {
  __shared__ f32x4 s_part[PA_NT];
  constexpr int TPR = BY_PAIR ? PA_NT : MG_WAVE;  // threads of a query head
  const int lane = threadIdx.x & (MG_WAVE - 1), tid = threadIdx.x % TPR;
  const int r = (int)mg_uniform(blockIdx.y * (PA_NT / TPR) + threadIdx.x / TPR);
  const int64_t pairs = (int64_t)a.Hk * a.tiles_q;
  int64_t steps, run;
  const int64_t all = pa_all<SPAN>(a, pairs, steps, run);
  const int shares = pa_shares_used(a, all);
  int64_t b, from;
  PaSeq seq;
  int pair, w0;
  if constexpr (BY_PAIR) {
    b = blockIdx.x / pairs, pair = (int)(blockIdx.x - b * pairs);
    seq = pa_seq_uniform<SPAN>(a, b);
    if (seq.steps == 0) return;
    from = (b ? pa_lane(steps, (int)b - 1) * pairs : 0) + (int64_t)pair * seq.steps;
    w0 = pa_holder(from, all, shares);
  } else {
    const int w = blockIdx.x + 1;
    if (w >= shares) return;
    const int64_t start = pa_share(w, all, shares);
    const PaPlace p = pa_find<SPAN>(a, pairs, steps, run, start);
    b = pa_uniform(p.b);
    seq = pa_seq_uniform<SPAN>(a, b);
    const PaPair at = pa_pair(start - p.before, seq.steps);
    if (at.step == 0) return;  // a pair starts here
    from = start - at.step, pair = at.pair, w0 = w - 1;
    if (pa_share(w0, all, shares) > from) return;  // an earlier start cuts it, too
  }
  const int hk = pair / a.tiles_q, tile_q = pair - hk * a.tiles_q;
  if (r >= a.rows || tile_q * PA_ROWS + r >= a.group) return;
  T* const dst = (T*)a.o + (b * a.H + hk * a.group + tile_q * PA_ROWS + r) * (int64_t)a.dv;
  const int n = pa_holder(from + seq.steps - 1, all, shares) - w0 + 1;
  if (n == 1) return;  // one share held it and has written it
  // The pieces are the first or second one of w0, then the first ones of w0 + 1 .. w0 + n - 1.
  const int second = pa_share(w0, all, shares) == from ? 0 : 1;
  const float2* const stat = (const float2*)(a.part + 2 * (int64_t)a.shares * a.rows * a.dv);
  auto place = [&](int i) { return ((int64_t)2 * (w0 + i) + (i ? 0 : second)) * a.rows + r; };
  // Threads side by side take four elements each, groups of them every n-th piece.  Each thread's
  // first pieces are on their way before the maximum is known.
  int wide = 1;
  while (4 * wide < a.dv) wide *= 2;
  const int groups = TPR / wide, mine = tid / wide, x = 4 * (tid - mine * wide);
  const bool whole = a.dv % 4 == 0 && x < a.dv;
  auto load = [&](int i) {
    const float* p = a.part + place(i < n ? i : 0) * a.dv;
    if (whole) return *(const f32x4*)(p + x);
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = p[x + e < a.dv ? x + e : 0];
    return v;
  };
  constexpr int AHEAD = BY_PAIR ? 16 : 4;
  f32x4 ahead[AHEAD];
  float peak[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) {
    const int i = mine + j * groups;
    ahead[j] = load(i);
    peak[j] = i < n ? stat[place(i)].x : -__builtin_inff();
  }
  // Each wave looks at all pieces' maxima and sums.
  float2 st = lane < n ? stat[place(lane)] : make_float2(-__builtin_inff(), 0.f);
  float top = st.x;
  for (int i = lane + MG_WAVE; i < n; i += MG_WAVE) top = fmaxf(top, stat[place(i)].x);
  top = pa_wave_max(top);
  const float base = top == -__builtin_inff() ? 0.f : top;
  float sum = pa_exp2(st.x - base) * st.y;
  for (int i = lane + MG_WAVE; i < n; i += MG_WAVE) {
    st = stat[place(i)];
    sum += pa_exp2(st.x - base) * st.y;
  }
  sum = mg_group_sum<64>(sum);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < AHEAD; ++j)
    if (mine + j * groups < n) v += pa_exp2(peak[j] - base) * ahead[j];
  for (int i = mine + AHEAD * groups; i < n; i += AHEAD * groups) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int at = i + j * groups;
      ahead[j] = load(at);
      peak[j] = at < n ? stat[place(at)].x : -__builtin_inff();
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (i + j * groups < n) v += pa_exp2(peak[j] - base) * ahead[j];
  }
  f32x4* const part = s_part + (threadIdx.x - tid);
  part[tid] = v;
  if constexpr (TPR == MG_WAVE) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
  if (mine == 0) {
    for (int j = 1; j < groups; ++j) v += part[j * wide + tid];
    const float inv = seq.bad ? __builtin_nanf("") : 1.f / sum;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (x + e < a.dv) dst[x + e] = pg_round<T>(v[e] * inv);
  }
}

// ---- host --------------------------------------------------------------------------------
// Shares: as many as the chip's 256 CUs hold workgroups at once.
int pa_most(int dk, int dv) { return 256 * pa_groups(dk > dv ? dk : dv, dv); }

bool pa_ok(int dtype, int64_t B, int H, int Hk, int dk, int dv, int64_t M, int64_t P) {
  return dtype >= 0 && dtype <= 2 && B >= 1 && H >= 1 && Hk >= 1 && H % Hk == 0 && dk >= 1 &&
         dv >= 1 && dk <= 256 && dv <= 256 && M >= 1 && P >= 1 && P < 1ll << 31 &&
         M < 1ll << 31 && M * P < (1ll << 31) - 1024 && B < 1ll << 24 && H < 1 << 24 &&
         B * H < 1ll << 24;
}
int pa_span(int dtype) { return dtype == 0 ? PaShape<float, 64, 64>::SPAN : PaShape<Bf16, 64, 64>::SPAN; }
// Workgroups: no more than there can be steps.
int pa_shares(int dtype, int64_t B, int H, int Hk, int dk, int dv, int64_t M, int64_t P) {
  const int64_t span = pa_span(dtype), tiles = (H / Hk + PA_ROWS - 1) / PA_ROWS;
  const int64_t per = (M * P + span - 1) / span * Hk * tiles;
  const int64_t most = pa_most(dk, dv);
  return (int)(per >= most || B >= most || per * B >= most ? most : per * B);
}
int pa_rows(int H, int Hk) { return H / Hk < PA_ROWS ? H / Hk : PA_ROWS; }

template <typename T, int DK, int DV>
void pa_launch(const PaArgs& a, hipStream_t stream) {
  // Vectors of a chunk: 16 bytes, 8 where a chunk is no more.
  const int e = sizeof(T), bk = DK * e / 16 < 16 ? 8 : 16, bv = DV * e / 16 < 16 ? 8 : 16;
  bool vec = a.dk * e % bk == 0 && a.dv * e % bv == 0 && ((uintptr_t)a.k & (bk - 1)) == 0 &&
             ((uintptr_t)a.v & (bv - 1)) == 0 && ((uintptr_t)a.q & (bk - 1)) == 0 &&
             a.qs[0] * e % bk == 0 && a.qs[1] * e % bk == 0;
  for (int i = 0; i < 3; ++i) vec = vec && a.ks[i] * e % bk == 0 && a.vs[i] * e % bv == 0;
  const dim3 grid(a.shares), nt(PA_NT);
  if (vec && a.P.d % 4 == 0)
    hipLaunchKernelGGL((paged_attention<T, DK, DV, true, true>), grid, nt, 0, stream, a);
  else if (vec)
    hipLaunchKernelGGL((paged_attention<T, DK, DV, true, false>), grid, nt, 0, stream, a);
  else
    hipLaunchKernelGGL((paged_attention<T, DK, DV, false, false>), grid, nt, 0, stream, a);
}
template <typename T>
int pa_run(const PaArgs& a, hipStream_t stream) {
  const int dk = a.dk > a.dv ? a.dk : a.dv;
  if (dk <= 64) pa_launch<T, 64, 64>(a, stream);
  else if (dk <= 128 && a.dv <= 64) pa_launch<T, 128, 64>(a, stream);
  else if (dk <= 128) pa_launch<T, 128, 128>(a, stream);
  else if (a.dv <= 128) pa_launch<T, 256, 128>(a, stream);
  else pa_launch<T, 256, 256>(a, stream);
  if (hipGetLastError() != hipSuccess) return MG_ERR_LAUNCH;
  // Where no pair can have two steps, or all are one share, none is cut.
  constexpr int SPAN = PaShape<T, 64, 64>::SPAN;
  if (a.shares == 1 || a.room <= SPAN) return MG_OK;
  // By pair where one has more than some eight pieces.  (64 x 4096 tokens, one key head, both
  // launches: 33 us by starts, 41 with a workgroup in a wave's place.  262144 tokens of one key head:
  // the join takes 26 us by starts, nearly all of which cut the same pair.)
  const int64_t all = a.B * a.Hk * a.tiles_q;
  if (all * 8 >= a.shares || a.B > MG_WAVE)
    hipLaunchKernelGGL((paged_attention_join<T, SPAN, false>),
                       dim3(a.shares - 1, (a.rows + PA_NW - 1) / PA_NW), dim3(PA_NT), 0, stream, a);
  else
    hipLaunchKernelGGL((paged_attention_join<T, SPAN, true>), dim3((unsigned)all, a.rows),
                       dim3(PA_NT), 0, stream, a);
  return hipGetLastError() == hipSuccess ? MG_OK : MG_ERR_LAUNCH;
}

}  // namespace

extern "C" {

size_t mg_paged_attention_workspace_bytes(int dtype, int64_t B, int H, int Hk, int dk, int dv,
                                          int64_t M, int64_t P) {
  if (!pa_ok(dtype, B, H, Hk, dk, dv, M, P)) return 0;
  return (size_t)2 * pa_shares(dtype, B, H, Hk, dk, dv, M, P) * pa_rows(H, Hk) * (dv + 2) * sizeof(float);
}

int mg_paged_attention_step(int dtype, const void* q, const void* k_cache, const void* v_cache,
                            const int64_t* strides, int ints, const void* pages,
                            const void* lengths, void* o, int64_t B, int H, int Hk, int dk, int dv,
                            int64_t N, int64_t M, int64_t P, int64_t window, float scale, void* ws,
                            size_t ws_bytes, hipStream_t stream) {
  if (!q || !k_cache || !v_cache || !strides || !pages || !lengths || !o || !ws || ints < 0 ||
      ints > 3 || N < 1 || N >= 1ll << 31 || window < 0 || !pa_ok(dtype, B, H, Hk, dk, dv, M, P))
    return MG_ERR_ARG;
  if (ws_bytes < mg_paged_attention_workspace_bytes(dtype, B, H, Hk, dk, dv, M, P))
    return MG_ERR_WORKSPACE;
  PaArgs a = {};
  a.q = q, a.k = k_cache, a.v = v_cache, a.o = o;
  a.pages = Ints{pages, ints & 1}, a.lengths = Ints{lengths, ints >> 1};
  a.qs[0] = strides[0], a.qs[1] = strides[1];
  for (int i = 0; i < 3; ++i) a.ks[i] = strides[2 + i], a.vs[i] = strides[5 + i];
  a.page_stride = strides[8];
  a.B = B, a.N = N, a.room = M * P, a.window = window, a.P = pg_divisor(P);
  a.H = H, a.Hk = Hk, a.group = H / Hk, a.tiles_q = (a.group + PA_ROWS - 1) / PA_ROWS;
  a.dk = dk, a.dv = dv;
  a.few_steps = B * (M * P / pa_span(dtype) + 2) < 1ll << 31;
  a.scale = scale * 1.4426950408889634f;
  a.shares = pa_shares(dtype, B, H, Hk, dk, dv, M, P), a.part = (float*)ws, a.rows = pa_rows(H, Hk);
  if (dtype == 0) return pa_run<float>(a, stream);
  return dtype == 1 ? pa_run<Bf16>(a, stream) : pa_run<Fp16>(a, stream);
}

}  // extern "C"
