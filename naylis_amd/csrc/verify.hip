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
// Weights and their sums are fp64: a token is a place among up to 152000
// cumulative sums, and an error of fp32's 2^-24 would move the border between two
// tokens of the tail past u once in a hundred draws.  fp64 runs at fp32's rate
// here, and 2^x costs ten products (a polynomial of degree 10 fitted at the
// Chebyshev nodes of [-1/2, 1/2], off by 3e-16).
//
// Three launches: a workgroup for each part of each row leaves (largest logit,
// its place, sum of 2^z against it) -- all that the rows' bytes are read for; a
// workgroup for each part of a row with a draft turned away sums its remaining
// weights (only with q); one for each sequence finds the part and the token in it.
// Each of the last two finds a by itself from the parts' sums, which lie in L2.
#include "common.h"
#include "launch.h"
#include "timing.h"

#include <algorithm>
#include <type_traits>

namespace naylis {

namespace {

constexpr int kStatThreads = 256;

// what the first launch leaves of a part of a row
struct VerifyStat {
  float top;   // largest logit
  int at;      // its first place
  double sum;  // of e^((x - top) / T), the draft's own token left out
};
static_assert(sizeof(VerifyStat) == 16, "the workspace is counted in these");

// 2^t for t <= 0: exact powers from the exponent's bits, 0 below 2^-1000, NaN for NaN
__device__ __forceinline__ double pow2(double t) {
  constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
  const double c = t < -1000.0 ? -1000.0 : t;
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
  const uint64_t b = __builtin_bit_cast(uint64_t, p);
  const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, shifted);
  const double r = __builtin_bit_cast(double, b + ((uint64_t)n << 52));
  return t < -1000.0 ? 0.0 : r;
}

// e^((x - top) / T), scale = log2(e) / T; 0 for x = -inf
__device__ __forceinline__ double weight(float x, float top, double scale) {
  return pow2(((double)x - (double)top) * scale);
}

__device__ __forceinline__ float load1(const bf16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ float load1(const float* p) { return *p; }

// Eight logits of a row, j0 .. j0 + 7, where j0 - shift is a multiple of 8: the
// row's 16-byte pieces of memory; -inf outside [0, V).
template <typename T>
__device__ __forceinline__ void load8(const T* row, long j0, int V, float (&x)[8]) {
  if (j0 >= 0 && j0 + 8 <= V) {
    if constexpr (sizeof(T) == 2) {
      const uint4 u = *reinterpret_cast<const uint4*>(row + j0);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
      const f32x4 a = *reinterpret_cast<const f32x4*>(row + j0), b = *reinterpret_cast<const f32x4*>(row + j0 + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = a[i];
        x[4 + i] = b[i];
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = j0 + i >= 0 && j0 + i < V ? load1(row + j0 + i) : -INFINITY;
}

// elements between the last 16-byte boundary and the row's first
template <typename T>
__device__ __forceinline__ int shift_of(const T* row) {
  return (int)(((uintptr_t)row & 15) / sizeof(T));
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
  return x;
}

__device__ __forceinline__ double scale_of(float t) { return 1.4426950408889634074 / (t > 0.f ? (double)t : 1.0); }

}  // namespace

__device__ __forceinline__ int verify_drafts_of(const VerifyArgs& a, int b) {
  return a.lens ? min(max(a.lens[b], 0), a.N) : a.N;
}
__device__ __forceinline__ float verify_temperature(const VerifyArgs& a, int b) { return a.temps ? a.temps[b] : a.temp; }

// grid (parts, N + 1, B).  PART logits, eight for a thread at a time.
template <typename T, int PART>
__global__ __launch_bounds__(kStatThreads) void verify_stat_kernel(VerifyArgs a, const T* __restrict__ logits,
                                                                   VerifyStat* __restrict__ stat) {
  constexpr int C = PART / (8 * kStatThreads), WAVES = kStatThreads / 64;
  __shared__ float tops[WAVES];
  __shared__ int ats[WAVES];
  __shared__ double sums[WAVES];
  const int part = blockIdx.x, i = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = verify_drafts_of(a, b);
  if (i > n) return;
  const T* row = logits + b * a.ldb + i * a.ldt;
  const double scale = scale_of(verify_temperature(a, b));
  const long draft = i < n ? a.drafts[(long)b * a.N + i] : -1;
  const long j0 = (long)part * PART - shift_of(row) + 8 * tid;
  float x[C][8];
#pragma unroll
  for (int c = 0; c < C; ++c) load8(row, j0 + 8 * kStatThreads * c, a.V, x[c]);
  float top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      top = fmaxf(top, x[c][e]);
      nan |= x[c][e] != x[c][e];
    }
  const float own = top;
  top = wave_allmax(top);
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) top = fmaxf(top, tops[w]);
  int at = 0x7fffffff;
  if (own == top)
#pragma unroll
    for (int c = C - 1; c >= 0; --c)
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (x[c][e] == top) at = (int)(j0 + 8 * kStatThreads * c + e);
  // a part of -inf alone adds nothing; a row with a NaN or +inf has no weights
  const float ref = top == -INFINITY ? 0.f : top;
  double s = 0.0;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double w = weight(x[c][e], ref, scale);
      s += j0 + 8 * kStatThreads * c + e == draft ? 0.0 : w;
    }
  if (nan || top == INFINITY) s = __builtin_nan("");
  at = wave_allmin_i32(at);
  s = wave_sum(s);
  if (lane == 0) {
    ats[wave] = at;
    sums[wave] = s;
  }
  __syncthreads();
  if (tid) return;
#pragma unroll
  for (int w = 1; w < WAVES; ++w) {
    at = min(at, ats[w]);
    s += sums[w];
  }
  stat[((long)b * (a.N + 1) + i) * a.parts + part] = VerifyStat{top, at, s};
}

namespace {

// a row's parts joined, by a wave: every lane gets it
struct RowStat {
  float top;
  int at;
  double sum;  // with the draft's token
};

// the draft's weight against the row's largest logit, 0 for an id that is none
struct DraftWeight {
  float x = 0.f;
  bool some = false;
  __device__ __forceinline__ double operator()(float top, double scale) const {
    return some ? weight(x, top, scale) : 0.0;
  }
};

template <typename T>
__device__ __forceinline__ RowStat join_row(const VerifyArgs& a, const VerifyStat* s, const T* row, long draft,
                                            double scale, double& dw) {
  const int lane = threadIdx.x & 63;
  DraftWeight d;
  if (draft >= 0 && draft < a.V) {
    d.x = load1(row + draft);
    d.some = true;
  }
  float top = -INFINITY;
  for (int p = lane; p < a.parts; p += 64) top = fmaxf(top, s[p].top);
  top = wave_allmax(top);
  const float ref = top == -INFINITY ? 0.f : top;
  int at = 0x7fffffff;
  double sum = 0.0;
  for (int p = lane; p < a.parts; p += 64) {
    const VerifyStat v = s[p];
    if (v.top == top) at = min(at, v.at);
    sum += v.top == -INFINITY ? v.sum : v.sum * weight(v.top, ref, scale);
  }
  dw = d(ref, scale);
  return RowStat{top, wave_allmin_i32(at), wave_sum(sum) + dw};
}

// What a sequence's decision is: drafts kept, and the row behind them.
struct Decision {
  int kept, n;
  RowStat row;
  double draft_weight;  // of the draft turned away
};

// By a whole workgroup; `red` and `out` in LDS.
template <typename T>
__device__ __forceinline__ Decision decide(const VerifyArgs& a, const T* logits, const VerifyStat* stat, int b,
                                           int* red, Decision* out) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
  const int n = verify_drafts_of(a, b);
  const float t = verify_temperature(a, b);
  const double scale = scale_of(t);
  if (tid == 0) *red = n;
  __syncthreads();
  const auto row_of = [&](int i) { return logits + b * a.ldb + i * a.ldt; };
  const auto stat_of = [&](int i) { return stat + ((long)b * (a.N + 1) + i) * a.parts; };
  for (int i = wave; i < n; i += waves) {
    const long d = a.drafts[(long)b * a.N + i];
    double dw;
    const RowStat r = join_row(a, stat_of(i), row_of(i), d, scale, dw);
    bool keep = false;
    if (d >= 0 && d < a.V) {
      const double u = a.uniforms[(long)b * (a.N + 1) + i];
      double q = 1.0;
      if (a.probs) {
        const long at = b * a.lqb + i * a.lqt + d;
        q = a.probs_bf16 ? bf16_to_f32(((const bf16_t*)a.probs)[at]) : ((const float*)a.probs)[at];
      }
      const double p = t > 0.f ? dw / r.sum : r.sum > 0.0 && r.at == d ? 1.0 : 0.0;
      keep = u * q < p;
    }
    if (!keep && lane == 0) atomicMin(red, i);
  }
  __syncthreads();
  const int kept = *red;
  if (wave == 0) {
    const long d = kept < n ? a.drafts[(long)b * a.N + kept] : -1;
    double dw;
    const RowStat r = join_row(a, stat_of(kept), row_of(kept), d, scale, dw);
    if (lane == 0) *out = Decision{kept, n, r, dw};
  }
  __syncthreads();
  return *out;
}

// The weights of eight tokens of the row behind the kept drafts: what is left of p.
template <typename T>
struct Left {
  const VerifyArgs& a;
  const T* row;
  const void* probs;  // q of the draft turned away, or NULL
  long without;       // a draft found by a rule that was turned away, or -1
  float top;
  int at;  // place of the largest logit
  double scale, inv;
  bool greedy;

  __device__ __forceinline__ void operator()(long j0, double (&w)[8]) const {
    float x[8];
    load8(row, j0, a.V, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const long j = j0 + e;
      w[e] = greedy ? (j == at ? 1.0 : 0.0) : weight(x[e], top, scale) * inv;
      if (probs) {
        double q = 0.0;
        if (j >= 0 && j < a.V) q = a.probs_bf16 ? bf16_to_f32(((const bf16_t*)probs)[j]) : ((const float*)probs)[j];
        const double r = w[e] - q;
        w[e] = r > 0.0 ? r : 0.0;
      } else if (j == without) {
        w[e] = 0.0;
      }
    }
  }
};

template <typename T>
__device__ __forceinline__ Left<T> left_of(const VerifyArgs& a, const T* logits, int b, const Decision& d, bool less) {
  const float t = verify_temperature(a, b);
  const T* row = logits + b * a.ldb + d.kept * a.ldt;
  const bool turned = less && d.kept < d.n;
  const void* probs = nullptr;
  if (turned && a.probs) {
    const long at = b * a.lqb + d.kept * a.lqt;
    probs = a.probs_bf16 ? (const void*)((const bf16_t*)a.probs + at) : (const void*)((const float*)a.probs + at);
  }
  const long without = turned && !a.probs ? a.drafts[(long)b * a.N + d.kept] : -1;
  return Left<T>{a, row, probs, without, d.row.top, d.row.at, scale_of(t), 1.0 / d.row.sum, !(t > 0.f)};
}

}  // namespace

// grid (parts, B), with q only: the sums of max(0, p - q) over the parts of a row
// whose draft was turned away.
template <typename T, int PART>
__global__ __launch_bounds__(kStatThreads) void verify_left_kernel(VerifyArgs a, const T* __restrict__ logits,
                                                                   const VerifyStat* __restrict__ stat,
                                                                   double* __restrict__ left) {
  __shared__ int red;
  __shared__ Decision dec;
  __shared__ double sums[kStatThreads / 64];
  const int part = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const Decision d = decide(a, logits, stat, b, &red, &dec);
  if (d.kept == d.n) return;
  const Left<T> l = left_of(a, logits, b, d, true);
  const long j0 = (long)part * PART - shift_of(l.row) + 8 * tid;
  double s = 0.0;
#pragma unroll 2
  for (int c = 0; c < PART / (8 * kStatThreads); ++c) {
    double w[8];
    l(j0 + 8 * kStatThreads * c, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += w[e];
  }
  s = wave_sum(s);
  if ((tid & 63) == 0) sums[tid >> 6] = s;
  __syncthreads();
  if (tid) return;
#pragma unroll
  for (int w = 1; w < kStatThreads / 64; ++w) s += sums[w];
  left[(long)b * a.parts + part] = s;
}

// grid (B), PART / 8 threads: the part that the random number falls in, the
// token in it, and the sequence's results.
template <typename T, int PART>
__global__ __launch_bounds__(PART / 8) void verify_pick_kernel(VerifyArgs a, const T* __restrict__ logits,
                                                               const VerifyStat* __restrict__ stat,
                                                               const double* __restrict__ left) {
  constexpr int WAVES = PART / 512;
  __shared__ int red, found, last;
  __shared__ Decision dec;
  __shared__ double sums[WAVES], before;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Decision d = decide(a, logits, stat, b, &red, &dec);
  const double u = a.uniforms[(long)b * (a.N + 1) + a.N];
  const bool greedy = !(verify_temperature(a, b) > 0.f), some = d.row.sum > 0.0;  // (not NaN)
  const VerifyStat* s = stat + ((long)b * (a.N + 1) + d.kept) * a.parts;
  long token = -1;
  if (greedy) {
    // what is left of a weight that is all on one token is on it too
    if (some) token = d.row.at;
  } else if (some) {
    // weight of a part: of what is left of p, or of p where that is nothing
    const bool turned = d.kept < d.n;
    const long gone = turned ? a.drafts[(long)b * a.N + d.kept] : -1;
    const Left<T> whole = left_of(a, logits, b, d, false);
    const int shift = shift_of(whole.row);
    const auto part_weight = [&](int p, bool less) {
      if (less && a.probs) return left[(long)b * a.parts + p];
      const VerifyStat v = s[p];
      double w = v.top == -INFINITY ? 0.0 : v.sum * weight(v.top, d.row.top, whole.scale);
      if (!less && turned && gone >= 0 && (gone + shift) / PART == p) w += d.draft_weight;
      return w * whole.inv;
    };
    bool less = turned;
    double total = 0.0;
    for (int p = lane; p < a.parts; p += 64) total += part_weight(p, less);
    total = wave_sum(total);
    if (less && !(total > 0.0)) {
      less = false;
      total = 0.0;
      for (int p = lane; p < a.parts; p += 64) total += part_weight(p, less);
      total = wave_sum(total);
    }
    const double target = u * total;
    // the first part whose cumulative weight passes the target, else the last with any
    int part = -1;
    double base = 0.0;
    for (int p0 = 0, done = 0; p0 < a.parts && !done; p0 += 64) {
      const int p = p0 + lane;
      const double own = p < a.parts ? part_weight(p, less) : 0.0;
      double sum = own;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const double y = __shfl_up(sum, o, 64);
        if (lane >= o) sum += y;
      }
      const unsigned long long past = __ballot(own > 0.0 && base + sum > target), any = __ballot(own > 0.0);
      const unsigned long long from = past ? past & -past : any ? 1ull << (63 - __clzll(any)) : 0;
      if (from) {
        const int l = __ffsll(from) - 1;
        part = p0 + l;
        before = base + __shfl(sum - own, l, 64);  // (the same in every thread)
      }
      done = past != 0;
      base += __shfl(sum, 63, 64);
    }
    if (tid == 0) {
      found = 0x7fffffff;
      last = -1;
    }
    __syncthreads();
    const double start = before;
    const Left<T> l = left_of(a, logits, b, d, less);
    const long j0 = (long)part * PART - shift + 8 * tid;
    double w[8], own = 0.0;
    l(j0, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) own += w[e];
    double sum = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(sum, o, 64);
      if (lane >= o) sum += y;
    }
    if (lane == 63) sums[wave] = sum;
    __syncthreads();
    double at = start + (sum - own);
    for (int v = 0; v < wave; ++v) at += sums[v];
    int hit = 0x7fffffff, mine = -1;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      at += w[e];
      if (w[e] > 0.0) {
        mine = (int)(j0 + e);
        if (at > target && hit == 0x7fffffff) hit = (int)(j0 + e);
      }
    }
    if (hit != 0x7fffffff) atomicMin(&found, hit);
    if (mine >= 0) atomicMax(&last, mine);
    __syncthreads();
    token = found != 0x7fffffff ? found : last;
  }
  for (int i = tid; i <= a.N; i += PART / 8)
    a.tokens[(long)b * (a.N + 1) + i] = i < d.kept ? a.drafts[(long)b * a.N + i] : i == d.kept ? token : -1;
  if (tid == 0) a.accepted[b] = d.kept;
}

namespace {

// Parts of 8192 logits where they fill the chip, else of 2048.
int verify_part(const VerifyArgs& a) {
  const long cells = (long)a.B * (a.N + 1) * a.V;
  return cells >= 8192l * 1024 ? 8192 : 2048;
}
// (a row that begins between two 16-byte boundaries may need one more)
int verify_parts(const VerifyArgs& a) { return (int)(((long)a.V + 7 + verify_part(a) - 1) / verify_part(a)); }

}  // namespace

size_t verify_ws_bytes(const VerifyArgs& a) {
  const size_t parts = verify_parts(a);
  return parts * a.B * (a.N + 1) * sizeof(VerifyStat) + (a.probs ? parts * a.B * sizeof(double) : 0);
}

hipError_t launch_verify(VerifyArgs a, const void* logits, bool bf16, void* ws, hipStream_t st) {
  a.parts = verify_parts(a);
  VerifyStat* stat = (VerifyStat*)ws;
  double* left = (double*)(stat + (size_t)a.parts * a.B * (a.N + 1));
  auto run = [&](auto type, auto part) {
    using T = decltype(type);
    constexpr int PART = decltype(part)::value;
    const T* x = (const T*)logits;
    NAYLIS_TIMED("verify_stat", st,
                 hipLaunchKernelGGL((verify_stat_kernel<T, PART>), dim3(a.parts, a.N + 1, a.B), dim3(kStatThreads), 0,
                                    st, a, x, stat));
    if (a.probs && a.N > 0) {
      NAYLIS_TIMED("verify_left", st,
                   hipLaunchKernelGGL((verify_left_kernel<T, PART>), dim3(a.parts, a.B), dim3(kStatThreads), 0, st, a,
                                      x, (const VerifyStat*)stat, left));
    }
    NAYLIS_TIMED("verify_pick", st,
                 hipLaunchKernelGGL((verify_pick_kernel<T, PART>), dim3(a.B), dim3(PART / 8), 0, st, a, x,
                                    (const VerifyStat*)stat, (const double*)left));
  };
  auto pick = [&](auto part) { bf16 ? run(bf16_t{}, part) : run(float{}, part); };
  verify_part(a) == 8192 ? pick(std::integral_constant<int, 8192>{}) : pick(std::integral_constant<int, 2048>{});
  return hipGetLastError();
}

}  // namespace naylis
