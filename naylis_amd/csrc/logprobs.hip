// Log probabilities of given tokens under rows of logits, each row's entropy
// and its likeliest tokens, and the gradient of the first two:
//   lse = log sum_j e^{x_j},  lp_j = x_j - lse,  p = e^lp,
//   logp = lp[token],  H = -sum_j p_j lp_j,
//   dx_j = g_logp (1[j = token] - p_j) - g_H p_j (lp_j + H).
// The reference keeps the summed loss of such rows (model.py:536-545).
//
// One workgroup per row (a few wide rows: one per part of a row, and a second
// launch that joins them), any V, any row stride and address: 16-byte chunks
// from the row's first 16-byte boundary, the few elements beside them one a
// thread.  Forward: one pass with a running reference m (the largest logit so
// far), s = sum 2^z and t = sum 2^z z, z the log2 of e^x over e^m, per thread; H =
// (log2 s - t / s) ln 2.  All statistics are fp32, saved as (m, log2 s, H): lp =
// (z - log2 s) ln 2 keeps the last bits that a single log-sum-exp would lose.
//
// The top k come from a second look at the row (registers, or the caches): the
// k-th largest of the threads' maxima is a value that at least k logits reach,
// and few others; those are collected in LDS and ranked (value, then lowest
// index).  Where too many reach it (a row of equal logits, or a mask that leaves
// fewer than k threads a finite one) k passes take one each: 64 x 32768 with ten
// allowed columns and the top 20 102 us (8.7), 4096 x 50001 1525 (127).
//
// Many rows are bound by HBM: 4096 x 50001 bf16 69 us (5.9 TB/s; fp32 127 us, 6.5
// TB/s), with the top 20, read twice, 122; a thread that keeps values as fp32
// between maximum and sum, 8 chunks at a time, takes 200 registers and 105 us.
// The gradient 143 to 154 us (5.3 to 5.7 TB/s read and written; a large copy 4.95).  Few rows
// are bound by the steps within a workgroup: 64 x 32768 with the top 20 8.9 us
// (1024 threads; 19.6 with 512 and a second read), of which 3 are launch and
// first load.  One row of 151999 in 8 parts 13.7 us, in one 21.9; 64 of them 17.4
// and 22.9.  Parts of 4096 columns of a 32768 row cost more than they save (9 + 6 us).
#include "common.h"
#include "launch.h"
#include "timing.h"

#include <algorithm>
#include <type_traits>

namespace naylis {

namespace {

constexpr int kCand = 1024;     // candidates ranked at once
constexpr int kMaxParts = 8;    // parts of a row
constexpr float kLn2 = 0.6931471805599453f;

// order of torch's descending sort as an unsigned key: NaN first, -0 equal to 0.
// No key is all ones: with column 0 that would make the rank key that stands
// for "before every logit".
__device__ __forceinline__ uint32_t sort_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x != x ? 0xfffffffeu : (u >> 31) ? ~u : u | 0x80000000u;
}

template <typename T>
__device__ __forceinline__ float value(T x) {
  if constexpr (sizeof(T) == 2)
    return bf16_to_f32(x);
  else
    return x;
}

// A row of V values: whole 16-byte chunks of E from the first 16-byte boundary
// on, and the few elements before and behind them, one for each of the first
// threads (`extra`).
template <typename T>
struct Row {
  static constexpr int E = 16 / sizeof(T);
  const T* x;
  int V, head, chunks;
  __device__ __forceinline__ Row(const T* p, int V_) : x(p), V(V_) {
    head = min((int)((16 - (uintptr_t)p % 16) % 16 / sizeof(T)), V);
    chunks = (V - head) / E;
  }
  __device__ __forceinline__ int first(int i) const { return head + E * i; }
  // the element outside the chunks that thread tid holds, or -1
  __device__ __forceinline__ int extra(int tid) const {
    const int j = tid < head ? tid : tid + E * chunks;
    return j < V && (tid < head || j >= head + E * chunks) ? j : -1;
  }
  template <bool ONCE>  // not read again: kept out of the caches' way
  __device__ __forceinline__ uint4 get(int i) const {
    const f32x4* p = reinterpret_cast<const f32x4*>(x + first(i));
    return __builtin_bit_cast(uint4, ONCE ? __builtin_nontemporal_load(p) : *p);
  }
  // U chunks i0, i0 + step, ..; those past the last are -inf
  template <int U, bool ONCE>
  __device__ __forceinline__ void get(uint4 (&u)[U], int i0, int step, bool all) const {
    if (all) {
#pragma unroll
      for (int i = 0; i < U; ++i) u[i] = get<ONCE>(i0 + i * step);
    } else {
      const uint32_t none = E == 8 ? 0xff80ff80u : 0xff800000u;
#pragma unroll
      for (int i = 0; i < U; ++i)
        u[i] = i0 + i * step < chunks ? get<ONCE>(i0 + i * step) : make_uint4(none, none, none, none);
    }
  }
};

// element e of a chunk
template <int E>
__device__ __forceinline__ float element(const uint4& u, int e) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  if constexpr (E == 4) return __uint_as_float(w[e]);
  return __uint_as_float((e & 1) ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
}

// max(a, b, c), NaN left out; written out because fmaxf of bits from memory
// costs a second instruction that quiets NaN
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// The reference of a sum of powers of two is its largest logit m, as c = m log2 e
// rounded once: all its terms x log2 e - c use the same c, so its rounding drops
// out.  Past 2^24 that rounding is more than an exponent may be off (and c can
// overflow): there the reference is m itself, and the terms are (x - m) log2 e.
constexpr float kFar = 16777216.f;
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) > kFar; }

// log2 of e^m over e^w for the references m and w, no less than -1e20 (finite
// times any sum)
__device__ __forceinline__ float ref_step(float m, float w) {
#pragma clang fp contract(off)
  const float c = m * kLog2e, cw = w * kLog2e;
  float d = c - cw;
  if (is_far(m) || is_far(w)) {
    d = is_far(m) ? is_far(w) ? (m - w) * kLog2e : fmaf(m, kLog2e, -cw) : -fmaf(w, kLog2e, -c);
    d = d < -1e20f ? -1e20f : d;
  }
  return d;
}

// log2 of e^x over e^m for the reference m (near: one within 2^24)
__device__ __forceinline__ float log2_near(float x, float m) {
  const float c = m * kLog2e;
  return fmaf(x, kLog2e, -c);
}
__device__ __forceinline__ float log2_ratio(float x, float m) {
  return is_far(m) ? (x - m) * kLog2e : log2_near(x, m);
}

// Sums of a part of a row against its largest x, m: s = sum 2^z, t = sum 2^z z
// with z the log2 of e^x over e^m.
struct Sums {
  float m, s, t;
  // against the reference of a whole; an empty part (m = -inf) weighs nothing
  __device__ __forceinline__ void rescale(float w) {
    const float d = ref_step(m, w), a = __builtin_amdgcn_exp2f(d);
    t = m == -INFINITY ? 0.f : a * fmaf(d, s, t);
    s = m == -INFINITY ? 0.f : a * s;
    m = w;
  }
};

// U chunks of a thread into its sums: per value a shift or mask, half a maximum,
// two fused multiply-adds, an exponential, a maximum and a sum
template <int E, int U>
__device__ __forceinline__ void add_chunks(Sums& a, const uint4 (&u)[U], bool& nan) {
  float m = a.m;
#pragma unroll
  for (int i = 0; i < U; ++i)
#pragma unroll
    for (int e = 0; e < E; e += 2) m = max3(m, element<E>(u[i], e), element<E>(u[i], e + 1));
  if (m == -INFINITY) {  // nothing but -inf (or NaN) so far
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) nan |= element<E>(u[i], e) != element<E>(u[i], e);
    return;
  }
  if (a.m == -INFINITY)
    a.m = m;
  else if (m > a.m)
    a.rescale(m);
  float s[2] = {a.s, 0.f}, t[2] = {a.t, 0.f};  // two chains
  auto add = [&](auto log2_of) {
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float z = log2_of(element<E>(u[i], e)), p = __builtin_amdgcn_exp2f(z);
        s[e & 1] += p;
        t[e & 1] = fmaf(p, fmaxf(z, -1e30f), t[e & 1]);  // 0 log 0 = 0
      }
  };
  if (__ballot(is_far(m)) == 0) {
    add([&](float x) { return log2_near(x, a.m); });
  } else {  // log2_ratio of both kinds of lanes in one form
    const float from = is_far(m) ? a.m : 0.f, c = is_far(m) ? 0.f : a.m * kLog2e;
    add([&](float x) { return fmaf(x - from, kLog2e, -c); });
  }
  a.s = s[0] + s[1];
  a.t = t[0] + t[1];
}

// one value more
__device__ __forceinline__ void add_one(Sums& a, float x, bool& nan) {
  nan |= x != x;
  if (!(x > -INFINITY)) return;
  if (a.m == -INFINITY)
    a.m = x;
  else if (x > a.m)
    a.rescale(x);
  const float z = log2_ratio(x, a.m), p = __builtin_amdgcn_exp2f(z);
  a.s += p;
  a.t = fmaf(p, fmaxf(z, -1e30f), a.t);
}

// The order of the top: a logit's sort key, then the lowest column.
__device__ __forceinline__ unsigned long long rank_key(float f, int j) {
  return ((unsigned long long)sort_key(f) << 32) | (uint32_t)~j;
}
__device__ __forceinline__ int column(unsigned long long k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float logit(unsigned long long k) {
  const uint32_t u = (uint32_t)(k >> 32);
  return __uint_as_float((u >> 31) ? u & 0x7fffffffu : ~u);
}

// log p of a logit from its row's reference and log2 of its sum; a far logit's in
// its own units, where its product with log2 e may overflow
__device__ __forceinline__ float log_prob(float x, float m, float ls) {
  return is_far(x) || is_far(m) ? (x - m) - ls * kLn2 : (log2_near(x, m) - ls) * kLn2;
}

// Joins the sums of `count` <= 64 parts that stand in LDS; every lane gets them.
__device__ __forceinline__ Sums join_parts(const float* m, const float* s, const float* t, int count) {
  const int lane = threadIdx.x & 63, i = min(lane, count - 1);
  Sums a{m[i], s[i], t[i]};
  a.rescale(wave_allmax(a.m));
  a.s = wave_allsum(lane < count ? a.s : 0.f);
  a.t = wave_allsum(lane < count ? a.t : 0.f);
  return a;
}

struct LogprobsOut {
  float* logp;
  float* entropy;
  float* stat;
  int64_t* top_ids;
  float* top_logp;
};

// A row's numbers from its sums (one thread); returns log2 s.  A row without a
// finite logit: m = -inf, NaN throughout.
__device__ __forceinline__ void write_row(const LogprobsOut& o, long r, const Sums& a, float ls, float xt, bool ignored,
                                          bool in_range) {
  const float ent = (ls - a.t / a.s) * kLn2;
  o.logp[r] = ignored ? 0.f : in_range ? log_prob(xt, a.m, ls) : __builtin_nanf("");
  o.entropy[r] = ent;
  if (o.stat) {
    o.stat[3 * r] = a.m;
    o.stat[3 * r + 1] = ls;
    o.stat[3 * r + 2] = ent;
  }
}

}  // namespace

// One row, or (parts > 1) one of its parts of `width` columns: then the sums
// and the part's `top` rank keys (0 behind its last) go to `part_sums` and
// `part_keys` for logprobs_join_kernel.
// HELD: a thread's U chunks are all there are and stay in registers, so that
// the second look (TOP) reads no memory; else they pass U at a time.
template <typename T, int NT, int U, bool HELD, bool TOP>
__global__ __launch_bounds__(NT) void logprobs_fwd_kernel(const T* __restrict__ logits, long ld,
                                                          const int64_t* __restrict__ tokens, LogprobsOut o, int V,
                                                          int top, long ignore_index, int parts, int width,
                                                          float* __restrict__ part_sums,
                                                          unsigned long long* __restrict__ part_keys) {
  constexpr int E = Row<T>::E, W = NT / 64;
  constexpr int RB = 4;       // key bits found in a round
  constexpr int VW = 16 / W;  // their values that a wave looks at
  constexpr int KEYBITS = sizeof(T) == 2 ? 16 : 32;
  static_assert(W == 16 || W == 4, "a power of four waves");
  __shared__ float red[3][W];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long r = blockIdx.x;
  const int col0 = blockIdx.y * width;  // the first column of this part
  const T* x = logits + r * ld;
  const Row<T> row(x + col0, min(width, V - col0));
  const long tok = parts == 1 ? tokens[r] : 0;
  const bool in_range = tok >= 0 && tok < V;
  const float xt = parts == 1 ? value(x[in_range ? tok : 0]) : 0.f;
  const int je = row.extra(tid);
  const float xe = je >= 0 ? value(row.x[je]) : -INFINITY;

  Sums a{-INFINITY, 0.f, 0.f};
  bool nan = false;
  uint4 u[U];
  if constexpr (HELD) {
    row.template get<U, !TOP>(u, tid, NT, NT * U <= row.chunks);
    add_chunks<E, U>(a, u, nan);
  } else {
    for (int c0 = 0; c0 < row.chunks; c0 += NT * U) {
      row.template get<U, !TOP>(u, c0 + tid, NT, c0 + NT * U <= row.chunks);
      add_chunks<E, U>(a, u, nan);
    }
  }
  add_one(a, xe, nan);
  const float mine = a.m;  // one of the logits, or -inf
  if (nan) a = Sums{0.f, __builtin_nanf(""), 0.f};
  a.rescale(wave_allmax(a.m));
  a.s = wave_allsum(a.s);
  a.t = wave_allsum(a.t);
  if (lane == 0) {
    red[0][wave] = a.m;
    red[1][wave] = a.s;
    red[2][wave] = a.t;
  }
  __syncthreads();
  a = join_parts(red[0], red[1], red[2], W);
  const float ls = log2f(a.s);
  const long part = r * parts + blockIdx.y;
  if (tid == 0) {
    if (parts == 1) {
      write_row(o, r, a, ls, xt, tok == ignore_index, in_range);
    } else {
      part_sums[3 * part] = a.m;
      part_sums[3 * part + 1] = a.s;
      part_sums[3 * part + 2] = a.t;
    }
  }
  if constexpr (TOP) {
    __shared__ uint32_t maxima[NT];
    __shared__ int counts[2][16];
    __shared__ unsigned long long cand[kCand];
    __shared__ int count;
    __shared__ unsigned long long best_s[W];
    maxima[tid] = sort_key(mine) >> (32 - KEYBITS);
    if (tid == 0) count = 0;
    __syncthreads();
    // the top-th largest of the threads' maxima, four bits of its key a round: the
    // waves count the maxima that reach the bits found so far and each next four
    uint32_t key[NT / 64], bound = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) key[i] = maxima[64 * i + lane];
#pragma unroll
    for (int shift = KEYBITS - RB, round = 0; shift >= 0; shift -= RB, ++round) {
#pragma unroll
      for (int v = 0; v < VW; ++v) {
        const uint32_t next = bound | ((uint32_t)(wave * VW + v) << shift);
        int n = 0;
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) n += __popcll(__ballot(key[i] >= next));
        if (lane == 0) counts[round & 1][wave * VW + v] = n;
      }
      __syncthreads();
      // the counts fall, so the last value that `top` maxima reach is how many such there are, less one
      const int w = __popcll(__ballot(lane < 16 && counts[round & 1][lane & 15] >= top)) - 1;
      bound |= (uint32_t)max(w, 0) << shift;
    }
    // that value: bf16's keys lack the low half, zeros in a positive number's and ones in a
    // negative one's.  -inf where fewer than `top` threads hold a larger logit: all are
    // collected then
    const float least = logit((unsigned long long)bound << (64 - KEYBITS) |
                              (KEYBITS == 16 && bound >> 15 == 0 ? 0xffffull << 32 : 0));
    const bool plain = a.s == a.s;  // no NaN, which a maximum leaves out
    auto collect = [&](float f, int j) {
      if (f < least) return;
      const int at = atomicAdd(&count, 1);
      if (at < kCand) cand[at] = rank_key(f, col0 + j);
    };
    if (je >= 0) collect(xe, je);
    auto look = [&](int c0) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int c = c0 + tid + i * NT;
        float most = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; e += 2) most = max3(most, element<E>(u[i], e), element<E>(u[i], e + 1));
        if (c < row.chunks && !(plain && most < least)) {
#pragma unroll
          for (int e = 0; e < E; ++e) collect(element<E>(u[i], e), row.first(c) + e);
        }
      }
    };
    if constexpr (HELD) {
      look(0);
    } else {
      for (int c0 = 0; c0 < row.chunks; c0 += NT * U) {
        row.template get<U, false>(u, c0 + tid, NT, c0 + NT * U <= row.chunks);
        look(c0);
      }
    }
    __syncthreads();
    const int n = count;
    auto write = [&](int rank, unsigned long long k) {
      if (parts == 1) {
        o.top_ids[r * top + rank] = column(k);
        o.top_logp[r * top + rank] = log_prob(logit(k), a.m, ls);
      } else {
        part_keys[part * top + rank] = k;
      }
    };
    if (parts > 1 && tid >= n && tid < top) write(tid, 0);
    if (n <= kCand) {
      for (int i = tid; i < n; i += NT) {
        const unsigned long long k = cand[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) rank += cand[j] > k;
        if (rank < top) write(rank, k);
      }
      return;
    }
    // one pass for each: the best logit behind the last one taken
    unsigned long long last = ~0ull;  // no logit's key
    for (int i = 0; i < top; ++i) {
      unsigned long long best = 0;
      const auto see = [&](float f, int j) {
        const unsigned long long k = rank_key(f, col0 + j);
        if (k < last && k > best) best = k;
      };
      if (je >= 0) see(xe, je);
      for (int c = tid; c < row.chunks; c += NT) {
        const uint4 v = row.template get<false>(c);
#pragma unroll
        for (int e = 0; e < E; ++e) see(element<E>(v, e), row.first(c) + e);
      }
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const unsigned long long k = __shfl_xor(best, o, 64);
        best = k > best ? k : best;
      }
      __syncthreads();
      if (lane == 0) best_s[wave] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < W; ++w) best = best_s[w] > best ? best_s[w] : best;
      last = best;
      if (tid == 0) write(i, best);
    }
  }
}

// A row from its parts.
template <typename T>
__global__ __launch_bounds__(256) void logprobs_join_kernel(const T* __restrict__ logits, long ld,
                                                            const int64_t* __restrict__ tokens, LogprobsOut o, int V,
                                                            int top, long ignore_index, int parts,
                                                            const float* __restrict__ part_sums,
                                                            const unsigned long long* __restrict__ part_keys) {
  __shared__ float red[3][kMaxParts];
  __shared__ unsigned long long cand[kMaxParts * kLogprobsMaxTop];
  const int tid = threadIdx.x;
  const long r = blockIdx.x;
  const long tok = tokens[r];
  const bool in_range = tok >= 0 && tok < V;
  const float xt = value(logits[r * ld + (in_range ? tok : 0)]);
  if (tid < 3 * parts) red[tid % 3][tid / 3] = part_sums[3 * r * parts + tid];
  const int n = parts * top;
  for (int i = tid; i < n; i += 256) cand[i] = part_keys[r * n + i];
  __syncthreads();
  const Sums a = join_parts(red[0], red[1], red[2], parts);
  const float ls = log2f(a.s);
  if (tid == 0) write_row(o, r, a, ls, xt, tok == ignore_index, in_range);
  for (int i = tid; i < n; i += 256) {
    const unsigned long long k = cand[i];
    if (k == 0) continue;  // behind a part's last logit
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += cand[j] > k;
    if (rank < top) {
      o.top_ids[r * top + rank] = column(k);
      o.top_logp[r * top + rank] = log_prob(logit(k), a.m, ls);
    }
  }
}

// d logits of a slab of `slab` chunks of a row (the first one takes the elements
// beside the chunks too); slabs of a row are neighbours in the grid, so that what
// is under way at a time lies together in memory.  4096 x 50001 bf16: 143 to 154 us by
// card (beside 154, a workgroup a row 183, of 1024 threads 157), fp32 287 (362); 300 x
// 151999 30 (53).  Slabs of 512 chunks: 160, 267, 35.  g_logp and g_entropy may be null (no
// gradient).
constexpr int kBwdChunks = 4;  // of a thread, loaded at once
template <typename T>
__global__ __launch_bounds__(256) void logprobs_bwd_kernel(const T* __restrict__ logits, long ld,
                                                           const int64_t* __restrict__ tokens,
                                                           const float* __restrict__ stat,
                                                           const float* __restrict__ g_logp, long gl_stride,
                                                           const float* __restrict__ g_entropy, long ge_stride,
                                                           T* __restrict__ dlogits, int V, long ignore_index, int slabs,
                                                           int slab) {
  constexpr int E = Row<T>::E;
  const long r = blockIdx.x / (unsigned)slabs;
  const int begin = blockIdx.x % (unsigned)slabs * slab;
  // chunks at the gradient's alignment (its rows are dense); the logits' may differ
  const Row<T> out(dlogits + r * (long)V, V);
  const T* x = logits + r * ld;
  const bool same = (uintptr_t)x % 16 == (uintptr_t)out.x % 16;
  const long tok = tokens[r];
  const float ref = stat[3 * r], ls = stat[3 * r + 1], ent = stat[3 * r + 2];
  const float gl = !g_logp || tok == ignore_index ? 0.f
                   : tok >= 0 && tok < V          ? g_logp[r * gl_stride]
                                                  : __builtin_nanf("");
  const float ge = g_entropy ? g_entropy[r * ge_stride] : 0.f;
  // z ln 2 = log p; 0 log 0 = 0 (the comparison keeps NaN)
  const auto grad = [&](float f, int j) {
    const float z = log2_ratio(f, ref) - ls, p = __builtin_amdgcn_exp2f(z);
    return (j == tok ? gl : 0.f) - p * fmaf(ge, fmaf(z < -1e3f ? -1e3f : z, kLn2, ent), gl);
  };
  T* dx = dlogits + r * (long)V;
  constexpr int U = kBwdChunks;
  const int end = min(out.chunks, begin + slab);
  const int je = begin == 0 ? out.extra(threadIdx.x) : -1;
  if (tok == ignore_index && ge == 0.f) {  // zeros, also where the row has no probabilities (-inf or NaN)
    for (int c = begin + threadIdx.x; c < end; c += 256)
      *reinterpret_cast<uint4*>(dx + out.first(c)) = make_uint4(0, 0, 0, 0);
    if (je >= 0) dx[je] = T(0);
    return;
  }
  for (int c0 = begin + threadIdx.x; c0 < end; c0 += 256 * U) {
    uint4 u[U];
    if (same) {
#pragma unroll
      for (int i = 0; i < U; ++i)
        u[i] = *reinterpret_cast<const uint4*>(x + out.first(min(c0 + 256 * i, end - 1)));
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int j0 = out.first(c0 + 256 * i);
      if (c0 + 256 * i >= end) break;
      float d[E];
      if (same) {
#pragma unroll
        for (int e = 0; e < E; ++e) d[e] = grad(element<E>(u[i], e), j0 + e);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) d[e] = grad(value(x[j0 + e]), j0 + e);
      }
      f32x4 o;
      if constexpr (E == 8) {
        bf16x8 h;
#pragma unroll
        for (int e = 0; e < E; ++e) h[e] = (__bf16)d[e];
        o = __builtin_bit_cast(f32x4, h);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = d[e];
      }
      __builtin_nontemporal_store(o, reinterpret_cast<f32x4*>(dx + j0));
    }
  }
  if (je >= 0) {
    const float d = grad(value(x[je]), je);
    if constexpr (E == 8)
      dx[je] = f32_to_bf16(d);
    else
      dx[je] = d;
  }
}

// A few wide rows are cut into parts, up to two workgroups a CU, and joined by
// a second launch.
static int logprobs_parts(long N, int V) {
  return V < 65536 ? 1 : (int)std::max(1L, std::min(512 / std::max(N, 1L), (long)kMaxParts));
}

size_t logprobs_ws_bytes(long N, int V, int top) {
  const int parts = logprobs_parts(N, V);
  return parts == 1 ? 0 : (size_t)N * parts * (8 * (size_t)top + 12);
}

hipError_t launch_logprobs_fwd(const void* logits, bool bf16, long ld, const int64_t* tokens, float* logp,
                               float* entropy, float* stat, int64_t* top_ids, float* top_logp, void* ws, long N,
                               int V, int top, long ignore_index, hipStream_t st) {
  const LogprobsOut o{logp, entropy, stat, top_ids, top_logp};
  const int parts = logprobs_parts(N, V);
  const int width = parts == 1 ? V : ((V + parts - 1) / parts + 63) / 64 * 64;
  auto* keys = (unsigned long long*)ws;
  auto* sums = (float*)(keys + (size_t)N * parts * top);
  auto run = [&](auto kernel, auto* x, int threads) {
    NAYLIS_TIMED("logprobs_fwd", st,
                 hipLaunchKernelGGL(kernel, dim3((unsigned)N, parts), dim3(threads), 0, st, x, ld, tokens, o, V, top,
                                    ignore_index, parts, width, sums, keys));
    return hipGetLastError();
  };
  auto pick = [&](auto* x, auto want) {
    typedef std::remove_const_t<std::remove_pointer_t<decltype(x)>> T;
    constexpr bool TOP = decltype(want)::value;
    const long chunks = (long)width * sizeof(T) / 16;
    if (chunks <= 256 * 4) return run(logprobs_fwd_kernel<T, 256, 4, true, TOP>, x, 256);
    if (N > 512) return run(logprobs_fwd_kernel<T, 256, 4, false, TOP>, x, 256);
    if (chunks <= 1024 * 4) return run(logprobs_fwd_kernel<T, 1024, 4, true, TOP>, x, 1024);
    return run(logprobs_fwd_kernel<T, 1024, 4, false, TOP>, x, 1024);
  };
  auto all = [&](auto* x) {
    typedef std::remove_const_t<std::remove_pointer_t<decltype(x)>> T;
    const hipError_t e = top > 0 ? pick(x, std::true_type{}) : pick(x, std::false_type{});
    if (e != hipSuccess || parts == 1) return e;
    NAYLIS_TIMED("logprobs_join", st,
                 hipLaunchKernelGGL(logprobs_join_kernel<T>, dim3((unsigned)N), dim3(256), 0, st, x, ld, tokens, o, V,
                                    top, ignore_index, parts, (const float*)sums, (const unsigned long long*)keys));
    return hipGetLastError();
  };
  return bf16 ? all((const bf16_t*)logits) : all((const float*)logits);
}

hipError_t launch_logprobs_bwd(const void* logits, bool bf16, long ld, const int64_t* tokens, const float* stat,
                               const float* g_logp, long gl_stride, const float* g_entropy, long ge_stride,
                               void* dlogits, long N, int V, long ignore_index, hipStream_t st) {
  auto run = [&](auto kernel, auto* x) {
    typedef std::remove_const_t<std::remove_pointer_t<decltype(x)>> T;
    const int chunks = std::max(V / Row<T>::E, 1);
    int slab = 256 * kBwdChunks;
    while (N * ((chunks + slab - 1) / slab) >= 1L << 24) slab *= 2;  // (a launch has under 2^32 threads)
    const int slabs = (chunks + slab - 1) / slab;
    NAYLIS_TIMED("logprobs_bwd", st,
                 hipLaunchKernelGGL(kernel, dim3((unsigned)(N * slabs)), dim3(256), 0, st, x, ld, tokens, stat, g_logp,
                                    gl_stride, g_entropy, ge_stride, (T*)dlogits, V, ignore_index, slabs, slab));
  };
  if (bf16)
    run(logprobs_bwd_kernel<bf16_t>, (const bf16_t*)logits);
  else
    run(logprobs_bwd_kernel<float>, (const float*)logits);
  return hipGetLastError();
}

}  // namespace naylis
