// New keys and values into a paged cache, rotated by their positions on the way (gfx950).
//
//   p = start_b + t;  (a, b) -> (a cos - b sin, b cos + a sin) with the angle p f_i
//   k_cache[page, h, p % P] = turned k;  v_cache[page, h, p % P] = v;  q_out = turned q
// where page = pages[b, p / P].
//
// Bound by memory: q, k and v are read and written once.  A workgroup takes a few tokens of a
// sequence, all their heads: the angles' sines and cosines are formed once a token, in LDS, and
// serve every head.  A thread moves units of 16 bytes, or two of them that turn together.
//
// Angles are products in fp64, reduced to a part of a turn there: at position 2^20 a product in
// fp32 is off by 2^-4 radians.  Sines and cosines of the reduced angle are fp32.
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
};

constexpr int AP_NT = 256;
constexpr int AP_TABLE = 2048;  // sine and cosine pairs of a workgroup's tokens in LDS
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

// VE elements are a unit: 16 bytes, or 1 where sizes, strides or pointers do not allow it.
template <typename T, int VE>
__global__ __launch_bounds__(AP_NT) void paged_append(ApArgs a) {
  __shared__ float2 s_turn[AP_TABLE];
  __shared__ ApPlace s_place[AP_MOST];
  const int64_t b = blockIdx.x / a.parts, part = blockIdx.x - b * a.parts;
  const int64_t t0 = part * a.tokens;
  const int64_t left = a.T - t0;
  const int count = (int)(left < a.tokens ? left : a.tokens);
  const int64_t start = a.start[b];
  if ((int)threadIdx.x < count) {
    const int64_t t = t0 + threadIdx.x, p = start + t;
    ApPlace at = {0, 0, AP_KEPT};
    if (a.lengths.p && t >= a.lengths[b]) {
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
  for (int i = threadIdx.x; i < count * a.n; i += AP_NT) {
    const int t = i / a.n, f = i - t * a.n;
    const double w = a.wide_freq ? ((const double*)a.freq)[f] : (double)((const float*)a.freq)[f];
    // In turns, of which whole ones do not matter.
    const double turns = (double)(start + t0 + t) * w * 0.15915494309189533577;
    float sin, cos;
    sincospif(2.f * (float)(turns - rint(turns)), &sin, &cos);
    s_turn[i] = make_float2(cos, sin);
  }
  __syncthreads();

  // A head's units: pairs of units that turn together (n elements each; neighbours turn within
  // a unit), then single ones.
  typedef ApVec<T, VE> V;
  const bool within = a.interleaved != 0;
  const int turning = within ? 2 * a.n / VE : a.n / VE;
  const int ku = turning + (a.dk - 2 * a.n) / VE, vu = a.dv / VE;
  const int qn = a.q ? a.H * ku : 0, kn = a.Hk * ku, all = qn + kn + a.Hk * vu;
  for (int64_t i = threadIdx.x; i < (int64_t)count * all; i += AP_NT) {
    const int t = (int)(i / all);
    int u = (int)(i - (int64_t)t * all);
    const ApPlace at = s_place[t];
    const bool query = u < qn;
    if (!query && at.kind != AP_KEPT) continue;
    const T* src;
    T* dst;
    if (!query && u >= qn + kn) {
      u -= qn + kn;
      const int h = u / vu, c = (u - h * vu) * VE;
      src = (const T*)a.v + b * a.vs[0] + (t0 + t) * a.vs[1] + h * a.vs[2] + c;
      dst = (T*)a.vc + at.v + h * a.vcs[1] + c;
      *(V*)dst = *(const V*)src;
      continue;
    }
    if (!query) u -= qn;
    const int h = u / ku;
    int c = u - h * ku;
    if (query) {
      src = (const T*)a.q + b * a.qs[0] + (t0 + t) * a.qs[1] + h * a.qs[2];
      dst = (T*)a.qo + ((b * a.T + t0 + t) * a.H + h) * a.dk;
    } else {
      src = (const T*)a.k + b * a.ks[0] + (t0 + t) * a.ks[1] + h * a.ks[2];
      dst = (T*)a.kc + at.k + h * a.kcs[1];
    }
    const bool turns = c < turning, two = turns && !within;
    c = turns ? c * VE : 2 * a.n + (c - turning) * VE;
    V x, y;
    if (at.kind == AP_PADDING || at.kind == AP_BAD) {  // a query's row of no place
      const T fill = pg_round<T>(at.kind == AP_BAD ? __builtin_nanf("") : 0.f);
#pragma unroll
      for (int e = 0; e < VE; ++e) x.e[e] = fill;
      *(V*)(dst + c) = x;
      if (two) *(V*)(dst + a.n + c) = x;
      continue;
    }
    x = *(const V*)(src + c);
    if (!turns) {
      *(V*)(dst + c) = x;
      continue;
    }
    const float2* turn = s_turn + t * a.n;
    if (two) {
      y = *(const V*)(src + a.n + c);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float2 w = turn[c + e];
        const float p = pg_float(x.e[e]), r = pg_float(y.e[e]);
        x.e[e] = pg_round<T>(p * w.x - r * w.y);
        y.e[e] = pg_round<T>(r * w.x + p * w.y);
      }
      *(V*)(dst + c) = x;
      *(V*)(dst + a.n + c) = y;
    } else if constexpr (VE > 1) {
#pragma unroll
      for (int e = 0; e < VE; e += 2) {
        const float2 w = turn[(c + e) / 2];
        const float p = pg_float(x.e[e]), r = pg_float(x.e[e + 1]);
        x.e[e] = pg_round<T>(p * w.x - r * w.y);
        x.e[e + 1] = pg_round<T>(r * w.x + p * w.y);
      }
      *(V*)(dst + c) = x;
    } else {  // one element a thread: its neighbour is read here and written by its own thread
      const float2 w = turn[c / 2];
      const float p = pg_float(x.e[0]), r = pg_float(src[c ^ 1]);
      *(dst + c) = pg_round<T>(c & 1 ? p * w.x + r * w.y : p * w.x - r * w.y);
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
  // Tokens of a workgroup: two rounds of its threads' units, as many angles as LDS holds.
  const int64_t heads = (int64_t)((a.q ? a.H : 0) + a.Hk) * a.dk + (int64_t)a.Hk * a.dv;
  const int64_t units = heads / (vec ? VE : 1);
  int64_t n = 2 * AP_NT / (units > 1 ? units : 1);
  if (n > AP_MOST) n = AP_MOST;
  if (a.n && n > AP_TABLE / a.n) n = AP_TABLE / a.n;
  if (n > a.T) n = a.T;
  if (n < 1) n = 1;
  a.tokens = (int)n;
  a.parts = (a.T + n - 1) / n;
  const int64_t grid = B * a.parts;
  if (grid >= 1ll << 24) return MG_ERR_TOO_LARGE;  // 2^32 threads
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
