// Verification of drafted tokens against a model's logits, from given random
// numbers.  For sequence b with drafts d_0 .. d_{n-1} drawn from q_0 .. q_{n-1},
// p_i = softmax(logits_i / T) and uniform numbers u:
//   draft i is kept while u_i q_i(d_i) < p_i(d_i); a = the number kept;
//   the token behind them is drawn from max(0, p_a - q_a) where draft a was
//   turned away, from p_n where none was: the first j whose cumulative weight
//   exceeds u_N of the whole.
// What comes out is distributed as p's own tokens, whatever q is.  Without q
// (drafts found by a rule) q_i(d_i) = 1, and the rest of p is p without d_a.
// T = 0: p is all on the largest logit, the first of equal ones.
//
// The weights of the row that a token is drawn from, and their sums, are fp64: the
// token is a place among up to 152000 cumulative sums, and an error of fp32's 2^-24
// would move the border between two tokens of the tail past u once in a hundred
// draws.  fp64 runs at fp32's rate here, and 2^x costs ten products (a polynomial of
// degree 10 fitted at the Chebyshev nodes of [-1/2, 1/2], off by 3e-16).  The sums
// that only decide which drafts are kept are fp32 wherever that token's row is summed
// again: with q, in three launches, and in one with two drafts or more.  They are off by
// less than 2^-19: a weight 2^-a of a part by three roundings of a (over 2048 logits 11 on
// average at most) and two of itself, a lane's sum of eight by seven.  u falls that near
// to p a few times in a million draws.
//
// Launches: (1) a wave for each 2048 logits of each row leaves (largest logit, its
// place, sum of 2^z against it) -- all that the rows' bytes are read for; (2) for
// each sequence the drafts kept, and over the row behind them the parts' fp64 sums
//   S = sum e,  and with q  R = sum max(0, e - S' q),  Q = sum of q where that is not 0,
// e = e^((x - top) / T) and S' the fp32 sum: what is left of p weighs R + (S' - S) Q,
// for S is so near to S' that only tokens that weigh next to nothing change sides.  Where
// p and q differ by no more than fp32's rounding (q the softmax of the same logits) these
// are all that is left: the part is then found among other tokens than the token in it, or
// the token in p where the part has none.  There a draft is turned away once in a million;
// (3) a workgroup for each sequence finds the part and the token in it.  Few logits
// and no q: (1) in fp64, and no (2).
//
// One sequence, three drafts of a rule, 32768 logits: 10 us, two launches whose waves
// wait for chains of loads (parts, draft, logit; part, token).  64 sequences, four
// drafts, 50001 logits, q fp32: 23 us, of which (1) 9.4 (32 MB), (2) 9.2 and (3) 5.4,
// each of them mostly a launch's start and end.  48, seven, 151999, q bf16: 40 us, (1)
// 19.7 (117 MB, 5.9 TB/s, and the vector units in use all the time: the weights by one
// multiply-add each take as long), (2) 14: the decisions' chains of loads, then some
// thirty fp64 operations a logit (vector units 69 %), (3) 5.6.  The two with fp32 logits:
// 27 and 61, (1) 11.7 and 41 (233 MB, 5.7 TB/s).
#include "common.h"
#include "launch.h"
#include "timing.h"

#include <algorithm>
#include <type_traits>

namespace naylis {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kPiece = 512;          // logits of a wave at a time, eight a lane
constexpr int kPieces = 4;           // pieces of a part: PIECES 4, or 1 where one workgroup does it all
constexpr int kLeftWaves = 8;         // of the second launch, which decides in each workgroup
constexpr int kSmallParts = 128, kSmallWaves = 16;  // the workgroup that does it all
// Weights up to these are none, those of -inf count as 2^-1000: of a part, and of a
// token, so much less that a part with a weight has a token with one.
constexpr double kNothing = 0x1p-900, kNoToken = 0x1p-920;

// what the first launch leaves of a part of a row
struct VerifyStat {
  float top;   // largest logit
  int at;      // its first place
  double sum;  // of e^((x - top) / T), the draft's own token left out
};
static_assert(sizeof(VerifyStat) == 16, "the workspace is counted in these");
// what the second leaves of a part of the row behind the kept drafts, against its largest logit
struct VerifyLeft {
  double sum, over;  // S (a turned away draft of a rule left out), R
  float q;           // Q
};

// 2^t for t <= 0, 2^-1000 and less as 2^-1000 (NaN too: callers look for those)
__device__ __forceinline__ double pow2(double t) {
  constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
  const double c = __builtin_fmax(t, -1000.0);
  const double shifted = c + kRound, f = c - (shifted - kRound);
  double p = 0x1.e6064532b85cep-28;
  p = __builtin_fma(p, f, 0x1.b675bd731322bp-24);
  p = __builtin_fma(p, f, 0x1.62bfd472702f4p-20);
  p = __builtin_fma(p, f, 0x1.ffcb5405401d9p-17);
  p = __builtin_fma(p, f, 0x1.4309130972597p-13);
  p = __builtin_fma(p, f, 0x1.5d87fe9d7ab38p-10);
  p = __builtin_fma(p, f, 0x1.3b2ab6fba1dcfp-7);
  p = __builtin_fma(p, f, 0x1.c6b08d703ce45p-5);
  p = __builtin_fma(p, f, 0x1.ebfbdff82c598p-3);
  p = __builtin_fma(p, f, 0x1.62e42fefa3a19p-1);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)(uint32_t)__builtin_bit_cast(uint64_t, shifted));
}

// e^((x - top) / T), scale = log2(e) / T; next to nothing, 2^-1000, for x = -inf
__device__ __forceinline__ double weight(float x, float top, double scale) {
  return pow2(((double)x - (double)top) * scale);
}

__device__ __forceinline__ float load1(const bf16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ float load1(const float* p) { return *p; }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Eight numbers of a row as they lie in memory.
template <typename T>
struct Raw8;
template <>
struct Raw8<bf16_t> {
  u32x4 u;
  __device__ __forceinline__ float operator[](int e) const {
    return __uint_as_float(e & 1 ? u[e >> 1] & 0xffff0000u : u[e >> 1] << 16);
  }
  __device__ __forceinline__ void set(int e, float x) {  // (x is a bf16)
    const uint32_t b = __float_as_uint(x);
    u[e >> 1] = e & 1 ? (u[e >> 1] & 0xffffu) | (b & 0xffff0000u) : (u[e >> 1] & 0xffff0000u) | (b >> 16);
  }
};
template <>
struct Raw8<float> {
  f32x4 f[2];
  __device__ __forceinline__ float operator[](int e) const { return f[e >> 2][e & 3]; }
  __device__ __forceinline__ void set(int e, float x) { f[e >> 2][e & 3] = x; }
};

// Numbers j0 .. j0 + 7 of a row one by one, `none` outside [0, V).
template <typename T>
__device__ __forceinline__ Raw8<T> ends8(const T* row, int j0, int V, float none) {
  Raw8<T> x = {};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = load1(row + min(max(j0 + e, 0), V - 1));
    x.set(e, j0 + e >= 0 && j0 + e < V ? y : none);
  }
  return x;
}

// Logits j0 .. j0 + 7 of a row, where j0 + shift_of(row) is a multiple of 8: the
// row's 16-byte pieces of memory; -inf outside [0, V).
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* row, int j0, int V) {
  if (j0 >= 0 && j0 + 8 <= V) return *reinterpret_cast<const Raw8<T>*>(row + j0);
  return ends8(row, j0, V, -INFINITY);
}

// A wave's share of a part: eight a lane from `first` on, for each of its pieces.
// Only a row's first and last part look at their ends.
template <int PIECES, typename T>
__device__ __forceinline__ void load_part(const T* row, int first, int V, Raw8<T> (&x)[PIECES]) {
  const int j0 = first + 8 * (int)(threadIdx.x & 63);
  if (first >= 0 && first + PIECES * kPiece <= V) {
#pragma unroll
    for (int c = 0; c < PIECES; ++c) x[c] = *reinterpret_cast<const Raw8<T>*>(row + j0 + 512 * c);
  } else {
#pragma unroll
    for (int c = 0; c < PIECES; ++c) x[c] = load8(row, j0 + 512 * c, V);
  }
}

__device__ __forceinline__ float max3(float a, float b, float c) {  // (without making NaNs quiet first)
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Eight numbers of a row at any address, 0 outside [0, V).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Any8 {
  Raw8<T> x;
};
template <typename T>
__device__ __forceinline__ Raw8<T> any8(const T* p) {
  return reinterpret_cast<const Any8<T>*>(p)->x;
}

// q, in either type, eight at a time; 0 outside [0, V) and without q.
struct Q8 {
  Raw8<float> f;
  __device__ __forceinline__ Q8(const void* probs, bool bf16, int j0, int V) : f{} {
    if (!probs) return;
    const bool inside = j0 >= 0 && j0 + 8 <= V;
    if (bf16) {
      const bf16_t* p = (const bf16_t*)probs;
      const Raw8<bf16_t> h = inside ? any8(p + j0) : ends8(p, j0, V, 0.f);
      f.f[0] = __builtin_bit_cast(f32x4, h.u);
      half = true;
    } else {
      const float* p = (const float*)probs;
      f = inside ? any8(p + j0) : ends8(p, j0, V, 0.f);
    }
  }
  // (converted where it is used: the load stays under way until then)
  __device__ __forceinline__ void widen() {
    if (!half) return;
    const Raw8<bf16_t> h{__builtin_bit_cast(u32x4, f.f[0])};
#pragma unroll
    for (int e = 0; e < 8; ++e) f.set(e, h[e]);
  }
  bool half = false;
};

// elements between the last 16-byte boundary and the row's first
template <typename T>
__device__ __forceinline__ int shift_of(const T* row) {
  return (int)(((uintptr_t)row & 15) / sizeof(T));
}

// a double from the lane that a DPP control names, 0 where there is none
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double dpp_f64(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)u, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double lane_of(double x, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane((int)u, lane), hi = __builtin_amdgcn_readlane((int)(u >> 32), lane);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
// inclusive sum over the lanes: within rows of 16 (row_shr 1, 2, 4, 8), then row 0
// into 1 and 2 into 3 (row_bcast 15), rows 0 and 1 into 2 and 3 (row_bcast 31)
__device__ __forceinline__ double wave_scan(double x) {
  x += dpp_f64<0x111>(x);
  x += dpp_f64<0x112>(x);
  x += dpp_f64<0x114>(x);
  x += dpp_f64<0x118>(x);
  x += dpp_f64<0x142, 0xa>(x);
  x += dpp_f64<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ double wave_sum(double x) { return lane_of(wave_scan(x), 63); }

// (0 at infinity: -inf times it is NaN, which weighs next to nothing as -inf does)
__device__ __forceinline__ double scale_of(float t) { return 1.4426950408889634074 / (t > 0.f ? (double)t : 1.0); }
// whether fp32 holds differences of logits that matter, and log2(e) / T
__device__ __forceinline__ bool ordinary(float t) { return !(t > 0.f) || (t > 0x1p-100f && t < 0x1p100f); }

}  // namespace

__device__ __forceinline__ int verify_drafts_of(const VerifyArgs& a, int b) {
  return a.lens ? min(max(a.lens[b], 0), a.N) : a.N;
}
__device__ __forceinline__ float verify_temperature(const VerifyArgs& a, int b) {
  return a.temps ? a.temps[b] : a.temp;
}

namespace {

// A part of row i of sequence b, by a wave.  EXACT: sums in fp64.
template <int PIECES, bool EXACT, typename T>
__device__ __forceinline__ VerifyStat stat_part(const VerifyArgs& a, const T* logits, int b, int i, int n, int part) {
  const int lane = threadIdx.x & 63;
  const T* row = logits + b * a.ldb + i * a.ldt;
  const int first = part * PIECES * kPiece - shift_of(row), j0 = first + 8 * lane;
  Raw8<T> x[PIECES];
  load_part(row, first, a.V, x);
  const float t = verify_temperature(a, b);
  const double scale = scale_of(t);
  const long draft = i < n ? a.drafts[(long)b * a.N + i] : -1;
  float top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int c = 0; c < PIECES; ++c)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      top = max3(top, x[c][e], x[c][e + 1]);
      if constexpr (EXACT) nan |= __builtin_isunordered(x[c][e], x[c][e + 1]);
    }
  const float own = top;
  top = wave_allmax(top);
  int at = 0x7fffffff;
  if (!(t > 0.f) && own == top)
#pragma unroll
    for (int c = PIECES - 1; c >= 0; --c)
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (x[c][e] == top) at = j0 + 512 * c + e;
  // the draft's own weight stays out: what is left without it is exact however small
  if (draft >= first && draft < first + PIECES * kPiece) {
#pragma unroll
    for (int c = 0; c < PIECES; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (j0 + 512 * c + e == (int)draft) {
          nan |= x[c][e] != x[c][e];
          x[c].set(e, -INFINITY);
        }
  }
  // a part of -inf alone adds nothing; a row with a NaN (which an fp32 sum keeps) or
  // +inf has no weights
  double s = 0.0;
  if (!(top == -INFINITY)) {
    if constexpr (EXACT) {
      // (a loop in code too, here and below: what runs once a wave waits for its
      // instructions longer than for its numbers)
#pragma unroll 1
      for (int c = 0; c < PIECES; ++c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s += weight(x[0][e], top, scale);
#pragma unroll
        for (int k = 1; k < PIECES; ++k) x[k - 1] = x[k];
      }
    } else {
      float sums[PIECES] = {};
      const auto sum = [&](auto exponent) {
#pragma unroll
        for (int c = 0; c < PIECES; ++c)
#pragma unroll
          for (int e = 0; e < 8; ++e) sums[c] += __builtin_amdgcn_exp2f(exponent(x[c][e]));
      };
      const float fs = (float)scale;
      if (ordinary(t)) {
        sum([&](float y) { return (y - top) * fs; });
      } else {
        // differences beyond fp32's largest number, or a scale beyond it (above 0 at
        // infinity, so that -inf stays what it is)
        const float before = t > 1.f ? 0x1p-4f : 1.f, after = t > 1.f ? 1.f : 0x1p64f, low = top * before;
        const float rest = (float)fmax(scale / ((double)before * after), 0x1p-149);
        sum([&](float y) { return (mul_rn(y, before) - low) * after * rest; });
      }
#pragma unroll
      for (int c = 0; c < PIECES; ++c) s += sums[c];
    }
  }
  if constexpr (!EXACT) {
    if (top == -INFINITY) {  // of nothing but -inf and NaNs
#pragma unroll
      for (int c = 0; c < PIECES; ++c)
#pragma unroll
        for (int e = 0; e < 8; e += 2) nan |= __builtin_isunordered(x[c][e], x[c][e + 1]);
    }
  }
  if (__any(nan) || top == INFINITY) s = __builtin_nan("");
  if (!(t > 0.f)) at = wave_allmin_i32(at);
  return VerifyStat{top, at, wave_sum(s)};
}

// a row's parts joined: every lane of the wave gets it
struct RowStat {
  float top;
  int at;
  double sum, draft;  // with the draft's weight, and that
};

// What a row's decision reads, all of it under way at once: 64 parts, the draft and
// what depends on it.
struct RowIn {
  VerifyStat first;
  long draft;
  float x, q, u;
  bool some;
};
template <typename T>
__device__ __forceinline__ RowIn read_row(const VerifyArgs& a, const T* logits, const VerifyStat* s, int b, int i) {
  const int lane = threadIdx.x & 63;
  RowIn r;
  r.draft = i < a.N ? a.drafts[(long)b * a.N + i] : -1;
  r.first = s[(long)i * a.parts + min(lane, a.parts - 1)];
  r.u = a.uniforms[(long)b * (a.N + 1) + i];
  r.some = r.draft >= 0 && r.draft < a.V;
  r.x = r.some ? load1(logits + b * a.ldb + i * a.ldt + r.draft) : -INFINITY;
  r.q = 1.f;
  if (r.some && a.probs) {
    const long j = b * a.lqb + i * a.lqt + r.draft;
    r.q = a.probs_bf16 ? bf16_to_f32(((const bf16_t*)a.probs)[j]) : ((const float*)a.probs)[j];
  }
  return r;
}
__device__ __forceinline__ RowStat join_row(const VerifyArgs& a, const VerifyStat* s, const RowIn& r, double scale,
                                            bool drafted) {
  const int lane = threadIdx.x & 63;
  float top = r.first.top;  // (a part twice where there are few)
  for (int p = lane + 64; p < a.parts; p += 64) top = fmaxf(top, s[p].top);
  top = wave_allmax(top);
  int at = 0x7fffffff;
  double sum = 0.0;
  for (int p = lane; p < a.parts; p += 64) {
    const VerifyStat v = p < 64 ? r.first : s[p];
    if (v.top == top) at = min(at, v.at);
    sum += v.sum * weight(v.top, top, scale);  // (0 for a part of -inf)
  }
  const double d = drafted && r.x > -INFINITY ? weight(r.x, top, scale) : 0.0;
  return RowStat{top, wave_allmin_i32(at), wave_sum(sum) + d, d};
}

// What a sequence's decision is: drafts kept of n, and the row behind them.
struct Decision {
  int kept, n;
  float t;
  long gone;  // the draft turned away, or -1
  RowStat row;
};

// By a workgroup of WAVES, each of which takes every WAVES-th row up to the first
// that keeps no draft.  s: the sequence's parts.
template <int WAVES, typename T>
__device__ __forceinline__ Decision decide(const VerifyArgs& a, const T* logits, const VerifyStat* s, int b) {
  __shared__ int ends[WAVES];
  __shared__ RowStat rows[WAVES];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // (rows behind the drafts are read here too, and do not count)
  RowIn r = read_row(a, logits, s, b, min(wave, a.N));
  const int n = verify_drafts_of(a, b);
  const float t = verify_temperature(a, b);
  const double scale = scale_of(t);
  int end = 0x7fffffff;
  RowStat row = {};
#pragma unroll 1
  for (int i = wave; i <= n; i += WAVES) {
    const RowIn next = read_row(a, logits, s, b, min(i + WAVES, a.N));
    row = join_row(a, s + (long)i * a.parts, r, scale, i < n);
    const bool likely = t > 0.f ? (double)r.u * (double)r.q * row.sum < row.draft
                                : row.sum > 0.0 && row.at == r.draft && (double)r.u * (double)r.q < 1.0;
    if (!(i < n && r.some && likely)) {
      end = i;
      break;
    }
    r = next;
  }
  if ((threadIdx.x & 63) == 0) {
    ends[wave] = end;
    rows[wave] = row;
  }
  __syncthreads();
  int kept = ends[0], of = 0;
#pragma unroll
  for (int v = 1; v < WAVES; ++v) {
    of = ends[v] < kept ? v : of;
    kept = min(kept, ends[v]);
  }
  return Decision{kept, n, t, kept < n ? a.drafts[(long)b * a.N + kept] : -1, rows[of]};
}

// The row behind the kept drafts, and what is taken from its weights.
template <typename T>
struct Behind {
  const VerifyArgs& a;
  const T* row;
  const void* probs;  // q of the draft turned away, or NULL
  long gone;          // that draft, or -1
  float top;
  double scale;

  __device__ __forceinline__ Behind(const VerifyArgs& a, const T* logits, int b, const Decision& d)
      : a(a), row(logits + b * a.ldb + d.kept * a.ldt), probs(nullptr), gone(d.gone), top(d.row.top),
        scale(scale_of(d.t)) {
    if (d.kept == d.n || !a.probs) return;
    const long at = b * a.lqb + d.kept * a.lqt;
    probs = a.probs_bf16 ? (const void*)((const bf16_t*)a.probs + at) : (const void*)((const float*)a.probs + at);
  }
  __device__ __forceinline__ Raw8<T> logits(int j0) const { return load8(row, j0, a.V); }
  // e of a token; next to nothing for columns of -inf and none
  __device__ __forceinline__ double operator()(float x) const { return weight(x, top, scale); }
};

// The fp64 sums over a part of the row behind the kept drafts, by a wave.
template <int PIECES, typename T>
__device__ __forceinline__ VerifyLeft left_part(const VerifyArgs& a, const T* logits, int b, const Decision& d,
                                                int part) {
  const int lane = threadIdx.x & 63;
  const Behind<T> r(a, logits, b, d);
  const int j0 = part * PIECES * kPiece - shift_of(r.row) + 8 * lane;
  double sum = 0.0, over = 0.0;
  float qs = 0.f;
  Raw8<T> x = r.logits(j0);
  Q8 q(r.probs, a.probs_bf16, j0, a.V);
#pragma unroll 1
  for (int c = 0; c < PIECES; ++c) {
    const int j = j0 + kPiece * c;
    const bool more = c + 1 < PIECES;
    const Raw8<T> nx = more ? r.logits(j + kPiece) : x;
    const Q8 nq = more ? Q8(r.probs, a.probs_bf16, j + kPiece, a.V) : q;
    if (!r.probs && r.gone >= j && r.gone < j + 8)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (j + e == (int)r.gone) x.set(e, -INFINITY);
    q.widen();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double w = r(x[e]), m = __builtin_fma(-d.row.sum, (double)q.f[e], w);
      sum += w;
      over += fmax(m, 0.0);
      qs += m > 0.0 ? q.f[e] : 0.f;
    }
    x = nx;
    q = nq;
  }
  return VerifyLeft{wave_sum(sum), wave_sum(over), wave_allsum(qs)};
}

// The token behind the kept drafts of a row with a distribution, by a workgroup:
// the part that the random number falls in, and the token in it, a piece for each of
// the first PIECES waves.  LEFT: from the fp64 sums of left_part (l), else
// from those of the first launch (s).  first: the lane's of the first 64 parts, read
// beside the decision.
template <bool LEFT, int PIECES, typename T>
__device__ __forceinline__ long pick(const VerifyArgs& a, const T* logits, int b, const Decision& d,
                                     const VerifyStat* s, const VerifyLeft* l, const VerifyLeft& first) {
  __shared__ int found[PIECES], last[PIECES];
  __shared__ double sums[PIECES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const double u = a.uniforms[(long)b * (a.N + 1) + a.N];
  const Behind<T> r(a, logits, b, d);
  const int shift = shift_of(r.row);
  const int gone_part = r.gone >= 0 && r.gone < a.V ? (int)((r.gone + shift) / (PIECES * kPiece)) : -1;
  const auto left_of = [&](int p) { return p < 64 ? first : l[p]; };  // of the lane's parts
  double S = 0.0;  // over the whole row, of the e that q is taken from
  if (r.probs) {
    for (int p = lane; p < a.parts; p += 64) S += left_of(p).sum;
    S = wave_sum(S);
  }
  // weight of a part: of what is left of p (less), or of p where that is nothing
  const auto part_weight = [&](int p, bool less) {
    if (less && r.probs) {
      const VerifyLeft v = left_of(p);
      return fmax(v.over + (d.row.sum - S) * v.q, 0.0);
    }
    double w;
    if constexpr (LEFT)
      w = left_of(p).sum;
    else
      w = s[p].sum * weight(s[p].top, d.row.top, r.scale);
    return !less && !r.probs && p == gone_part ? w + d.row.draft : w;
  };
  const auto sum_of = [&](bool less) {
    double w = 0.0;
    for (int p = lane; p < a.parts; p += 64) w += part_weight(p, less);
    return wave_sum(w);
  };
  bool less = d.kept < d.n;
  // (again from all of p where less is none of it, or only what rounding left: a part
  // then has a weight of 1e-14 of p that none of its tokens has)
#pragma unroll 1
  for (;;) {
    const double total = sum_of(less);
    if (less && !(total > kNothing)) {
      less = false;
      continue;
    }
    const double target = u * total;
    // the first part whose cumulative weight passes the target, else the last with
    // any; every wave finds it by itself
    int part = -1;
    double base = 0.0, start = 0.0;
    for (int p0 = 0, done = 0; p0 < a.parts && !done; p0 += 64) {
      const int p = p0 + lane;
      const double own = p < a.parts ? part_weight(p, less) : 0.0, sum = wave_scan(own);
      const unsigned long long past = __ballot(own > kNothing && base + sum > target), any = __ballot(own > kNothing);
      const unsigned long long from = past ? past & -past : any ? 1ull << (63 - __clzll(any)) : 0;
      if (from) {
        const int at = __ffsll(from) - 1;
        part = p0 + at;
        start = base + lane_of(sum - own, at);
      }
      done = past != 0;
      base += lane_of(sum, 63);
    }
    double w[8], own = 0.0, sum = 0.0;
    const int j0 = part * PIECES * kPiece - shift + 8 * tid;
    if (wave < PIECES) {
      const Raw8<T> x = r.logits(j0);
      Q8 q(less ? r.probs : nullptr, a.probs_bf16, j0, a.V);
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = less && j0 + e == r.gone && !r.probs ? 0.0 : r(x[e]);
      if (less && r.probs) {
        q.widen();
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = fmax(__builtin_fma(-S, (double)q.f[e], w[e]), 0.0);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) own += w[e];
      sum = wave_scan(own);
      if (lane == 63) sums[wave] = sum;
    }
    __syncthreads();
    if (wave < PIECES) {
      double at = start + (sum - own);
      for (int v = 0; v < wave; ++v) at += sums[v];
      int hit = 0x7fffffff, mine = -1;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        at += w[e];
        if (w[e] > kNoToken) {
          mine = j0 + e;
          if (at > target && hit == 0x7fffffff) hit = j0 + e;
        }
      }
      const unsigned long long hits = __ballot(hit != 0x7fffffff), any = __ballot(mine >= 0);
      const int to = any ? __builtin_amdgcn_readlane(mine, 63 - __clzll(any)) : -1;
      const int from = hits ? __builtin_amdgcn_readlane(hit, __ffsll(hits) - 1) : 0x7fffffff;
      if (lane == 0) {
        found[wave] = from;
        last[wave] = to;
      }
    }
    __syncthreads();
    int from = 0x7fffffff, to = -1;
#pragma unroll
    for (int v = 0; v < PIECES; ++v) {
      from = min(from, found[v]);
      to = max(to, last[v]);
    }
    const int token = from != 0x7fffffff ? from : to;
    if (token >= 0 || !less) return token;
    less = false;
  }
}

// a row without a distribution, or greedy: no token, or the largest logit (what is
// left of a weight that is all on one token is on it too)
__device__ __forceinline__ bool drawn(const Decision& d) { return d.t > 0.f && d.row.sum > 0.0; }
__device__ __forceinline__ long undrawn(const Decision& d) { return d.row.sum > 0.0 ? d.row.at : -1; }

// a sequence's results, by a workgroup
__device__ __forceinline__ void answer(const VerifyArgs& a, int b, const Decision& d, long token) {
  for (int i = threadIdx.x; i <= a.N; i += blockDim.x)
    a.tokens[(long)b * (a.N + 1) + i] = i < d.kept ? a.drafts[(long)b * a.N + i] : i == d.kept ? token : -1;
  if (threadIdx.x == 0) a.accepted[b] = d.kept;
}

}  // namespace

// grid (parts / 4, N + 1, B), a part for each wave.  (Eight waves a SIMD have registers
// for a part of bf16 logits; the sums in fp64, and fp32 logits, which wait for memory, are
// left what they take: 74 and 50.)
template <typename T, bool EXACT>
__global__ __launch_bounds__(kThreads, EXACT || sizeof(T) == 4 ? 1 : 8) void verify_stat_kernel(
    VerifyArgs a, const T* __restrict__ logits, VerifyStat* __restrict__ stat) {
  const int i = blockIdx.y, b = blockIdx.z;
  const int part = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = verify_drafts_of(a, b);
  if (i > n || part >= a.parts) return;
  const VerifyStat s = stat_part<kPieces, EXACT>(a, logits, b, i, n, part);
  if ((threadIdx.x & 63) == 0) stat[((long)b * (a.N + 1) + i) * a.parts + part] = s;
}

// grid (parts / 8, B): the drafts kept, and the fp64 sums over the row behind them.
// (The last workgroup of a sequence finding the token here, behind a fence of the
// device, takes 6 us more than a launch of its own.)
template <typename T>
__global__ __launch_bounds__(64 * kLeftWaves) void verify_left_kernel(VerifyArgs a, const T* __restrict__ logits,
                                                               const VerifyStat* __restrict__ stat,
                                                               VerifyLeft* __restrict__ left,
                                                               Decision* __restrict__ decisions) {
  const int b = blockIdx.y;
  const int part = blockIdx.x * kLeftWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Decision d = decide<kLeftWaves>(a, logits, stat + (long)b * (a.N + 1) * a.parts, b);
  if (blockIdx.x == 0 && threadIdx.x == 0) decisions[b] = d;
  if (!drawn(d) || part >= a.parts) return;
  const VerifyLeft l = left_part<kPieces>(a, logits, b, d, part);
  if ((threadIdx.x & 63) == 0) left[(long)b * a.parts + part] = l;
}

// grid (B): the token, from the fp64 sums of the second launch (LEFT) or the first.
template <typename T, bool LEFT>
__global__ __launch_bounds__(kThreads) void verify_pick_kernel(VerifyArgs a, const T* __restrict__ logits,
                                                               const VerifyStat* __restrict__ stat,
                                                               const VerifyLeft* __restrict__ left,
                                                               const Decision* __restrict__ decisions) {
  const int b = blockIdx.x;
  Decision d;
  VerifyLeft first = {};
  left += (long)b * a.parts;
  if constexpr (LEFT) {
    first = left[min((int)threadIdx.x & 63, a.parts - 1)];
    d = decisions[b];
  } else {
    d = decide<kWaves>(a, logits, stat + (long)b * (a.N + 1) * a.parts, b);
  }
  const VerifyStat* s = stat + ((long)b * (a.N + 1) + d.kept) * a.parts;
  answer(a, b, d, drawn(d) ? pick<LEFT, kPieces>(a, logits, b, d, s, left, first) : undrawn(d));
}

// grid (B): all of it by one workgroup, where a sequence has few logits.  EXACT: without
// q, the rows' sums in fp64, so that there are no others to form.
template <typename T, bool EXACT>
__global__ __launch_bounds__(64 * kSmallWaves) void verify_small_kernel(VerifyArgs a, const T* __restrict__ logits) {
  __shared__ VerifyStat stat[kSmallParts];
  __shared__ VerifyLeft left[EXACT ? 1 : kSmallParts];
  const int b = blockIdx.x, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = verify_drafts_of(a, b);
  for (int k = wave; k < (n + 1) * a.parts; k += kSmallWaves) {
    const VerifyStat s = stat_part<1, EXACT>(a, logits, b, k / a.parts, n, k % a.parts);
    if (lane == 0) stat[k] = s;
  }
  __syncthreads();
  const Decision d = decide<kSmallWaves>(a, logits, stat, b);
  if (!drawn(d)) {
    answer(a, b, d, undrawn(d));
    return;
  }
  if constexpr (EXACT) {
    answer(a, b, d, pick<false, 1>(a, logits, b, d, stat + d.kept * a.parts, left, VerifyLeft{}));
  } else {
    for (int p = wave; p < a.parts; p += kSmallWaves) {
      const VerifyLeft l = left_part<1>(a, logits, b, d, p);
      if (lane == 0) left[p] = l;
    }
    __syncthreads();
    answer(a, b, d, pick<true, 1>(a, logits, b, d, stat, left, left[min(lane, a.parts - 1)]));
  }
}

namespace {

// (a row that begins between two 16-byte boundaries may need one more)
int verify_parts(const VerifyArgs& a, int pieces) {
  return (int)(((long)a.V + 7 + pieces * kPiece - 1) / (pieces * kPiece));
}

// One launch for sequences of few logits: its 16 waves pass N + 1 rows' parts and, in
// fp64, one row's, which takes twice as long a part (or both at once, up to one draft
// without q).  Beyond the limits a workgroup's CU is slower than launches over the chip
// (16 sequences, us in one launch and in more: without q, no drafts, 10000 logits 9.1 and
// 9.7; one, 7000 10.5 and 11.2, 8500 11.8 and 10.7; three, 3500 10.1 and 11.0, 5000 11.7
// and 11.1; with q, one draft, 14000 14.6 and 16.1, 23000 20.0 and 15.8; seven, 3500 13.1
// and 15.4, 5000 15.9 and 15.9).  Two launches, the first in fp64, where q is not given
// and the logits are few; else three.
enum VerifyForm { kSmall, kBrief, kFull };
VerifyForm verify_form(const VerifyArgs& a) {
  if ((long)verify_parts(a, 1) * (a.N + 3) <= (a.probs ? 112 : a.N <= 1 ? 60 : 50)) return kSmall;
  return !a.probs && (long)a.B * (a.N + 1) * a.V <= (1l << 24) ? kBrief : kFull;
}

}  // namespace

size_t verify_ws_bytes(const VerifyArgs& a) {
  const size_t parts = verify_parts(a, kPieces);
  const size_t stat = parts * a.B * (a.N + 1) * sizeof(VerifyStat);
  const VerifyForm form = verify_form(a);
  return form == kSmall ? 0 : form == kBrief ? stat : stat + a.B * (parts * sizeof(VerifyLeft) + sizeof(Decision));
}

hipError_t launch_verify(VerifyArgs a, const void* logits, bool bf16, void* ws, hipStream_t st) {
  const VerifyForm form = verify_form(a);
  a.parts = verify_parts(a, form == kSmall ? 1 : kPieces);
  VerifyStat* stat = (VerifyStat*)ws;
  VerifyLeft* left = (VerifyLeft*)(stat + (size_t)a.parts * a.B * (a.N + 1));
  Decision* decisions = (Decision*)(left + (size_t)a.parts * a.B);
  const unsigned groups = (a.parts + kWaves - 1) / kWaves;
  auto run = [&](auto type) {
    using T = decltype(type);
    const T* x = (const T*)logits;
    auto first = [&](auto exact) {
      NAYLIS_TIMED("verify_stat", st,
                   hipLaunchKernelGGL((verify_stat_kernel<T, decltype(exact)::value>), dim3(groups, a.N + 1, a.B),
                                      dim3(kThreads), 0, st, a, x, stat));
    };
    auto last = [&](auto from_left) {
      NAYLIS_TIMED("verify_pick", st,
                   hipLaunchKernelGGL((verify_pick_kernel<T, decltype(from_left)::value>), dim3(a.B), dim3(kThreads),
                                      0, st, a, x, (const VerifyStat*)stat, (const VerifyLeft*)left,
                                      (const Decision*)decisions));
    };
    if (form == kSmall) {
      auto all = [&](auto kernel) {
        NAYLIS_TIMED("verify_small", st,
                     hipLaunchKernelGGL(kernel, dim3(a.B), dim3(64 * kSmallWaves), 0, st, a, x));
      };
      // (an fp64 sum over two rows costs less than one more pass over one: without drafts,
      // 16 sequences of 5000 logits 8.4 us and 9.3, with one 9.4 and 9.8, with two level)
      !a.probs && a.N <= 1 ? all(verify_small_kernel<T, true>) : all(verify_small_kernel<T, false>);
    } else if (form == kBrief) {
      first(std::true_type{});
      last(std::false_type{});
    } else {
      first(std::false_type{});
      NAYLIS_TIMED("verify_left", st,
                   hipLaunchKernelGGL((verify_left_kernel<T>), dim3((a.parts + kLeftWaves - 1) / kLeftWaves, a.B),
                                      dim3(64 * kLeftWaves), 0, st, a, x,
                                      (const VerifyStat*)stat, left, decisions));
      last(std::true_type{});
    }
  };
  bf16 ? run(bf16_t{}) : run(float{});
  return hipGetLastError();
}

}  // namespace naylis
