// New keys and values into a paged cache, rotated by their positions on the way (gfx950).
//
//   p = start_b + t;  (a, b) -> (a cos - b sin, b cos + a sin) with the angle p f_i
//   k_cache[page, h, p % P] = turned k;  v_cache[page, h, p % P] = v;  q_out = turned q
// where page = pages[b, p / P].
//
// Bound by memory: q, k and v are read and written once.  A workgroup takes a few tokens of a
// sequence, all their heads: the angles' sines and cosines are formed once a token, in LDS, and
// serve every head.  A thread moves units of 16 bytes, or two of them that turn together, the
// same ones of one token after another: what they are and where they lie is worked out once, not
// for each (which took more of the vector units' time than the memory's).
//
// Angles are products in fp64, reduced to an eighth of a turn at most there: at position 2^20 a
// product in fp32 is off by 2^-4 radians, one in fp64 by 2^-33.  Sines and cosines of the rest are fp32.
//
// 16 x 2048 ragged tokens of 16 and 8 heads of 128 in bf16: 67 us, 5.2 TB/s with the padding's zeros.
#include "mg_paged.h"

namespace {

struct ApArgs {
  const void *q, *k, *v;
  void *kc, *vc, *qo;
  Ints pages, start, lengths;  // lengths.p may be null
  const void* freq;            // fp32, or fp64 where wide_freq; null without rotation
  int wide_freq, interleaved;
  int64_t qs[3], ks[3], vs[3];  // strides in elements: sequence, token, head
  int64_t kcs[3], vcs[3];       // page, head, slot
  int64_t page_stride;          // between the sequences' rows of pages
  int64_t T, N, M;
  int64_t parts;                // workgroups of a sequence
  int P, H, Hk, dk, dv, n;      // n: frequencies
  int tokens;                   // of a workgroup
  // units: of a head of q and k and of v (ku, vu), those of them that turn, of all q, of all k,
  // of a token
  int turning, ku, vu, qn, kn, all;
  int abreast;                  // tokens that the workgroup's threads take at a time
};

constexpr int AP_NT = 256;
constexpr int AP_TABLE = 1024;  // sine and cosine pairs of a workgroup's tokens in LDS
constexpr int AP_MOST = 16;     // tokens of a workgroup

template <typename T, int VE>
struct alignas(sizeof(T) * VE) ApVec {
  T e[VE];
};

// Where a token goes: the offsets of its rows in the caches without the head, or not at all.
struct ApPlace {
  int64_t k, v;
  int kind;
};
enum { AP_PADDING = 0, AP_KEPT = 1, AP_DROPPED = 2, AP_BAD = 3 };

template <typename T, int VE>
__device__ __forceinline__ void ap_get(const ApVec<T, VE>& v, float (&f)[VE]) {
#pragma unroll
  for (int e = 0; e < VE; ++e) f[e] = pg_float(v.e[e]);
}
template <typename T, int VE>
__device__ __forceinline__ void ap_set(ApVec<T, VE>& v, const float (&f)[VE]) {
  if constexpr (sizeof(T) == 2 && VE > 1) {
    unsigned w[VE / 2];
#pragma unroll
    for (int e = 0; e < VE; e += 2) w[e / 2] = pg_pack<T>(f[e], f[e + 1]);
    v = __builtin_bit_cast(ApVec<T, VE>, w);
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) v.e[e] = pg_round<T>(f[e]);
  }
}

// Past the caches: 75 us with ordinary stores in place of 67 at 16 x 2048 tokens.
template <typename T, int VE>
__device__ __forceinline__ void ap_store(T* to, const ApVec<T, VE>& v) {
  if constexpr (sizeof(v) == 16)
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), (u32x4*)to);
  else
    *(ApVec<T, VE>*)to = v;
}

// VE elements are a unit: 16 bytes, or 1 where sizes, strides or pointers do not allow it.
template <typename T, int VE>
__global__ __launch_bounds__(AP_NT) void paged_append(ApArgs a) {
  __shared__ alignas(16) float2 s_turn[AP_TABLE];
  __shared__ ApPlace s_place[AP_MOST];
  typedef ApVec<T, VE> V;
  const int64_t b = blockIdx.x / a.parts, part = blockIdx.x - b * a.parts;
  const int64_t t0 = part * a.tokens;
  const int count = (int)(a.T - t0 < a.tokens ? a.T - t0 : a.tokens);
  int live = count;  // tokens that are there
  if (a.lengths.p) {
    const int64_t n = a.lengths[b];
    live = n <= t0 ? 0 : (n - t0 < count ? (int)(n - t0) : count);
  }
  {
    const int64_t start = a.start[b];
    if ((int)threadIdx.x < count) {
      const int64_t p = start + t0 + threadIdx.x;
      ApPlace at = {0, 0, AP_KEPT};
      if ((int)threadIdx.x >= live) {
        at.kind = AP_PADDING;
      } else if (p < 0 || p / a.P >= a.M) {
        at.kind = AP_BAD;
      } else {
        const int64_t row = p / a.P, slot = p - row * a.P, page = a.pages[b * a.page_stride + row];
        at.kind = page < 0 ? AP_DROPPED : (page >= a.N ? AP_BAD : AP_KEPT);
        at.k = page * a.kcs[0] + slot * a.kcs[2];
        at.v = page * a.vcs[0] + slot * a.vcs[2];
      }
      s_place[threadIdx.x] = at;
    }
    for (int i = threadIdx.x; i < live * a.n; i += AP_NT) {
      const int t = i / a.n, f = i - t * a.n;
      const double w = a.wide_freq ? ((const double*)a.freq)[f] : (double)((const float*)a.freq)[f];
      // In quarter turns: the nearest whole number of them, modulo 4, and the rest, an eighth of a turn
      // at most either way.
      const double quarters = (double)(start + t0 + t) * w * 0.63661977236758134308;
      const double whole = rint(quarters);
      float sin, cos;
      sincospif(0.5f * (float)(quarters - whole), &sin, &cos);
      const int quadrant = (int)(whole - 4.0 * floor(0.25 * whole));
      const float c = quadrant & 1 ? sin : cos, s = quadrant & 1 ? cos : sin;
      s_turn[i] = make_float2(quadrant == 1 || quadrant == 2 ? -c : c, quadrant & 2 ? -s : s);
    }
  }
  __syncthreads();

  // A head's units: pairs of units that turn together (n elements each; neighbours turn within
  // a unit), then single ones.
  const int lead = a.abreast > 1 ? (int)threadIdx.x / a.all : 0;
  if (lead >= a.abreast) return;
  for (int i = (int)threadIdx.x - lead * a.all; i < a.all; i += AP_NT) {
    const bool query = i < a.qn, value = i >= a.qn + a.kn;
    const int j = query ? i : (value ? i - a.qn - a.kn : i - a.qn);
    const int h = j / (value ? a.vu : a.ku), in = j - h * (value ? a.vu : a.ku);
    const bool turns = !value && in < a.turning, two = turns && !a.interleaved;
    const int c = value || turns ? in * VE : 2 * a.n + (in - a.turning) * VE;
    const T* src;
    T* dst;
    int64_t step;
    if (query) {
      src = (const T*)a.q + b * a.qs[0] + h * a.qs[2], step = a.qs[1];
      dst = (T*)a.qo + ((b * a.T + t0) * a.H + h) * a.dk;
    } else if (value) {
      src = (const T*)a.v + b * a.vs[0] + h * a.vs[2], step = a.vs[1];
      dst = (T*)a.vc + h * a.vcs[1];
    } else {
      src = (const T*)a.k + b * a.ks[0] + h * a.ks[2], step = a.ks[1];
      dst = (T*)a.kc + h * a.kcs[1];
    }
    src += t0 * step + c, dst += c;
    const int64_t row = (int64_t)a.H * a.dk;
    // The other half of what turns: n elements on, or (one element a unit) the neighbour, which its
    // own thread writes.
    const int other = two ? a.n : (VE == 1 && turns ? (c & 1 ? -1 : 1) : 0);
    for (int t = lead; t < count; t += a.abreast) {
      V x, y;
      if (t < live) {  // padding is not read
        x = *(const V*)(src + t * step);
        if (other) y = *(const V*)(src + t * step + other);
      }
      const int kind = s_place[t].kind;
      if (!query && kind != AP_KEPT) continue;
      T* const to = dst + (query ? t * row : (value ? s_place[t].v : s_place[t].k));
      if (turns && t < live) {
        float p[VE], q[VE];
        ap_get(x, p), ap_get(y, q);
        const float2* const turn = s_turn + t * a.n;
        if (two) {
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const float2 w = turn[c + e];
            const float s = p[e] * w.x - q[e] * w.y;
            q[e] = q[e] * w.x + p[e] * w.y, p[e] = s;
          }
          ap_set(y, q);
        } else if constexpr (VE > 1) {
#pragma unroll
          for (int e = 0; e < VE; e += 2) {
            const float2 w = turn[(c + e) / 2];
            const float s = p[e] * w.x - p[e + 1] * w.y;
            p[e + 1] = p[e + 1] * w.x + p[e] * w.y, p[e] = s;
          }
        } else {
          const float2 w = turn[c / 2];
          p[0] = c & 1 ? p[0] * w.x + q[0] * w.y : p[0] * w.x - q[0] * w.y;
        }
        ap_set(x, p);
      }
      if (kind == AP_PADDING || kind == AP_BAD) {  // a query's row of no place
        float f[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) f[e] = kind == AP_BAD ? __builtin_nanf("") : 0.f;
        ap_set(x, f);
        y = x;
      }
      ap_store(to, x);
      if (two) ap_store(to + a.n, y);
    }
  }
}

bool ap_aligned(const void* p, const int64_t* strides, int bytes) {
  if ((uintptr_t)p & 15) return false;
  for (int i = 0; i < 3; ++i)
    if ((strides[i] * bytes) & 15) return false;
  return true;
}

template <typename T>
int ap_run(ApArgs& a, int64_t B, hipStream_t stream) {
  constexpr int VE = 16 / sizeof(T);
  const int e = sizeof(T);
  const bool vec = a.dk % VE == 0 && a.dv % VE == 0 &&
                   (a.interleaved ? 2 * a.n % VE == 0 : a.n % VE == 0) &&
                   (!a.q || (ap_aligned(a.q, a.qs, e) && ((uintptr_t)a.qo & 15) == 0)) &&
                   ap_aligned(a.k, a.ks, e) && ap_aligned(a.v, a.vs, e) &&
                   ap_aligned(a.kc, a.kcs, e) && ap_aligned(a.vc, a.vcs, e);
  if (B >= 1ll << 24 || a.T >= 1ll << 38) return MG_ERR_TOO_LARGE;
  const int ve = vec ? VE : 1;
  a.turning = (a.interleaved ? 2 * a.n : a.n) / ve;
  a.ku = a.turning + (a.dk - 2 * a.n) / ve, a.vu = a.dv / ve;
  a.qn = a.H * a.ku, a.kn = a.Hk * a.ku, a.all = a.qn + a.kn + a.Hk * a.vu;
  a.abreast = a.all < AP_NT ? AP_NT / a.all : 1;
  // Tokens of a workgroup: as many as leave the chip's 256 CUs 32 workgroups each, and as many
  // angles as LDS holds.  (16 x 2048 ragged tokens of 16 and 8 heads of 128 in bf16: 67 us, with 64
  // workgroups each 72, with 8 82.)
  int64_t n = a.abreast * ((B * a.T) / (8192 * (int64_t)a.abreast));
  if (n < a.abreast) n = a.abreast;
  if (n > AP_MOST) n = AP_MOST;
  if (a.n && n > AP_TABLE / a.n) n = AP_TABLE / a.n;
  if (n > a.T) n = a.T;
  if (a.abreast > n) a.abreast = (int)n;
  a.tokens = (int)n;
  a.parts = (a.T + n - 1) / n;
  const int64_t grid = B * a.parts;
  if (a.parts >= 1ll << 24 || grid >= 1ll << 24) return MG_ERR_TOO_LARGE;  // 2^32 threads
  if (vec)
    hipLaunchKernelGGL((paged_append<T, VE>), dim3((unsigned)grid), dim3(AP_NT), 0, stream, a);
  else
    hipLaunchKernelGGL((paged_append<T, 1>), dim3((unsigned)grid), dim3(AP_NT), 0, stream, a);
  return hipGetLastError() == hipSuccess ? MG_OK : MG_ERR_LAUNCH;
}

}  // namespace

extern "C" int mg_paged_append(int dtype, const void* q, const void* k, const void* v,
                               void* k_cache, void* v_cache, void* q_out, const int64_t* strides,
                               int ints, const void* pages, const void* start, const void* lengths,
                               int freq_dtype, const void* freq, int n, int interleaved, int64_t B,
                               int64_t T, int H, int Hk, int dk, int dv, int64_t N, int64_t M,
                               int64_t P, hipStream_t stream) {
  if (dtype < 0 || dtype > 2 || !k || !v || !k_cache || !v_cache || !strides || !pages || !start ||
      (q && !q_out) || ints < 0 || ints > 7 || B < 1 || T < 1 || Hk < 1 || dk < 1 || dv < 1 ||
      (q && H < 1) || N < 1 || M < 1 || P < 1 || P >= 1ll << 31 || T >= 1ll << 40 ||
      B >= 1ll << 40 || n < 0 || 2 * (int64_t)n > dk || (n && !freq) || (freq_dtype & ~1) ||
      n > AP_TABLE || (int64_t)Hk * dk + (int64_t)Hk * dv + (q ? (int64_t)H * dk : 0) >= 1ll << 26)
    return MG_ERR_ARG;
  ApArgs a = {};
  a.q = q, a.k = k, a.v = v, a.kc = k_cache, a.vc = v_cache, a.qo = q_out;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = strides[i], a.ks[i] = strides[3 + i], a.vs[i] = strides[6 + i];
    a.kcs[i] = strides[9 + i], a.vcs[i] = strides[12 + i];
  }
  a.page_stride = strides[15];
  a.pages = Ints{pages, ints & 1}, a.start = Ints{start, ints >> 1 & 1};
  a.lengths = Ints{lengths, ints >> 2 & 1};
  a.freq = freq, a.wide_freq = freq_dtype, a.interleaved = interleaved != 0 && n > 0;
  a.T = T, a.N = N, a.M = M, a.P = (int)P;
  a.H = q ? H : 0, a.Hk = Hk, a.dk = dk, a.dv = dv, a.n = n;
  if (dtype == 0) return ap_run<float>(a, B, stream);
  return dtype == 1 ? ap_run<Bf16>(a, B, stream) : ap_run<Fp16>(a, B, stream);
}
