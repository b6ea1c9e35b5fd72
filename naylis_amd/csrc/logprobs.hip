// Log probabilities of given tokens under rows of logits, each row's entropy
// and its likeliest tokens, and the gradient of the first two:
//   lse = log sum_j e^{x_j},  lp_j = x_j - lse,  p = e^lp,
//   logp = lp[token],  H = -sum_j p_j lp_j,
//   dx_j = g_logp (1[j = token] - p_j) - g_H p_j (lp_j + H).
// The reference keeps the summed loss of such rows (model.py:536-545).
//
// One workgroup per row, any V, any row stride and address: 16-byte chunks at
// the row's own alignment, its two ragged ends element by element.  Forward:
// one pass with a running maximum m, sum of e^{x - m} and sum of
// e^{x - m} (x - m) per thread, joined at the end; H = log s - t / s.  Bound by
// HBM (the logits once).  Statistics are fp32, saved as (m, log s, H): x - m is
// nearly exact where their sum would lose the last bits of small lp.
//
// The top k come from a second look at the row, out of the caches: the k-th
// largest of the threads' maxima is a value that at least k logits reach, and
// few others; those are collected in LDS and ranked (value, then lowest index).
// Where too many reach it (a row of equal logits) k passes take one each.
#include "common.h"
#include "launch.h"
#include "timing.h"

#include <type_traits>

namespace naylis {

namespace {

constexpr int kCand = 1024;  // candidates ranked at once

// order of torch's descending sort as an unsigned key: NaN first, -0 equal to 0
__device__ __forceinline__ uint32_t sort_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x != x ? 0xffffffffu : (u >> 31) ? ~u : u | 0x80000000u;
}

template <typename T>
__device__ __forceinline__ float value(T x) {
  if constexpr (sizeof(T) == 2)
    return bf16_to_f32(x);
  else
    return x;
}

// A row of V values in 16-byte chunks of E, counted from the 16-byte boundary
// at or before it: chunk i holds elements E i - skip .. E i - skip + E - 1.
template <typename T>
struct Row {
  static constexpr int E = 16 / sizeof(T);
  const T* x;
  int V, skip, chunks;
  __device__ __forceinline__ Row(const T* p, int V_) : x(p), V(V_) {
    skip = (int)((uintptr_t)p % 16 / sizeof(T));
    chunks = (V + skip + E - 1) / E;
  }
  // chunk i as fp32; elements outside the row (and chunks past it) are -inf
  __device__ __forceinline__ void get(int i, float (&f)[E]) const {
    const int j0 = E * i - skip;
    if (j0 >= 0 && j0 + E <= V) {
      const uint4 u = __builtin_bit_cast(uint4, *reinterpret_cast<const f32x4*>(x + j0));
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (E == 8) {
          f[2 * e] = __uint_as_float(w[e] << 16);
          f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        } else {
          f[e] = __uint_as_float(w[e]);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = j0 + e >= 0 && j0 + e < V ? value(x[j0 + e]) : -INFINITY;
    }
  }
};

// (m, s, t) of two parts of a row
struct Sums {
  float m, s, t;
  __device__ __forceinline__ void join(const Sums& o) {
    const float mn = fmaxf(m, o.m);
    const float da = m - mn, db = o.m - mn;  // -inf parts are empty: weight 0
    const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(da * kLog2e);
    const float b = o.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(db * kLog2e);
    t = (m == -INFINITY ? 0.f : a * fmaf(da, s, t)) + (o.m == -INFINITY ? 0.f : b * fmaf(db, o.s, o.t));
    s = a * s + b * o.s;
    m = mn;
  }
};

}  // namespace

template <typename T, int NT>
__global__ __launch_bounds__(NT) void logprobs_fwd_kernel(const T* __restrict__ logits, long ld,
                                                          const int64_t* __restrict__ tokens,
                                                          float* __restrict__ logp, float* __restrict__ entropy,
                                                          float* __restrict__ stat, int64_t* __restrict__ top_ids,
                                                          float* __restrict__ top_logp, int V, int top,
                                                          long ignore_index) {
  constexpr int E = Row<T>::E, W = NT / 64, U = 4;
  __shared__ Sums red[W];
  __shared__ float maxima[NT];
  __shared__ uint32_t cand_key[kCand];
  __shared__ int cand_id[kCand];
  __shared__ int count;
  __shared__ uint32_t bound_s;
  __shared__ unsigned long long best_s[W];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long r = blockIdx.x;
  const Row<T> row(logits + r * ld, V);
  const long tok = tokens[r];
  const bool in_range = tok >= 0 && tok < V;
  const float xt = value(row.x[in_range ? tok : 0]);

  Sums a{-INFINITY, 0.f, 0.f};
  bool nan = false;
  for (int c0 = tid; c0 < row.chunks; c0 += NT * U) {
    float f[U][E];
#pragma unroll
    for (int u = 0; u < U; ++u) row.get(c0 + u * NT, f[u]);
    float m = a.m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) m = fmaxf(m, f[u][e]);
    if (m == -INFINITY) {  // nothing but -inf (or NaN) so far
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) nan |= f[u][e] != f[u][e];
      continue;
    }
    if (a.m != -INFINITY) {
      const float da = a.m - m, al = __builtin_amdgcn_exp2f(da * kLog2e);
      a.t = al * fmaf(da, a.s, a.t);
      a.s *= al;
    }
    a.m = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = f[u][e] - m, p = __builtin_amdgcn_exp2f(d * kLog2e);
        a.s += p;
        a.t = fmaf(p, fmaxf(d, -1e30f), a.t);  // 0 log 0 = 0
      }
  }
  if (top > 0) maxima[tid] = a.m;  // a logit of the row, or -inf
  if (nan) {
    a.s = __builtin_nanf("");
    if (a.m == -INFINITY) a.m = 0.f;
  }
  // the wave's lanes, then the waves
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    Sums b{__shfl_xor(a.m, o, 64), __shfl_xor(a.s, o, 64), __shfl_xor(a.t, o, 64)};
    a.join(b);
  }
  if (lane == 0) red[wave] = a;
  if (tid == 0) count = 0;
  __syncthreads();
  a = red[0];
#pragma unroll
  for (int i = 1; i < W; ++i) a.join(red[i]);
  const float ls = logf(a.s);  // a row without a finite logit: m = -inf, log 0, NaN below
  if (tid == 0) {
    const float ent = ls - a.t / a.s;
    logp[r] = tok == ignore_index ? 0.f : in_range ? (xt - a.m) - ls : __builtin_nanf("");
    entropy[r] = ent;
    if (stat) {
      stat[3 * r] = a.m;
      stat[3 * r + 1] = ls;
      stat[3 * r + 2] = ent;
    }
  }
  if (top == 0) return;

  // the k-th largest of the threads' maxima, bit by bit from the top
  if (wave == 0) {
    uint32_t key[NT / 64];
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) key[i] = sort_key(maxima[64 * i + lane]);
    uint32_t bound = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t next = bound | (1u << bit);
      int n = 0;
#pragma unroll
      for (int i = 0; i < NT / 64; ++i) n += __popcll(__ballot(key[i] >= next));
      if (n >= top) bound = next;
    }
    if (lane == 0) bound_s = bound;
  }
  __syncthreads();
  const uint32_t bound = bound_s;
  for (int c0 = tid; c0 < row.chunks; c0 += NT * U) {
    float f[U][E];
#pragma unroll
    for (int u = 0; u < U; ++u) row.get(c0 + u * NT, f[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int j = E * (c0 + u * NT) - row.skip + e;
        if (sort_key(f[u][e]) >= bound && j >= 0 && j < V) {
          const int at = atomicAdd(&count, 1);
          if (at < kCand) {
            cand_key[at] = sort_key(f[u][e]);
            cand_id[at] = j;
          }
        }
      }
  }
  __syncthreads();
  int64_t* ids = top_ids + r * top;
  float* lps = top_logp + r * top;
  const int n = count;
  if (n <= kCand) {
    for (int i = tid; i < n; i += NT) {
      const uint32_t k = cand_key[i];
      const int id = cand_id[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += cand_key[j] > k || (cand_key[j] == k && cand_id[j] < id);
      if (rank < top) {
        ids[rank] = id;
        lps[rank] = (value(row.x[id]) - a.m) - ls;
      }
    }
    return;
  }
  // one pass for each: the best logit behind the last one taken
  unsigned long long last = ~0ull;  // key, then the lowest index first
  for (int i = 0; i < top; ++i) {
    unsigned long long best = 0;
    for (int c = tid; c < row.chunks; c += NT) {
      float f[E];
      row.get(c, f);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int j = E * c - row.skip + e;
        if (j < 0 || j >= V) continue;
        const unsigned long long k = ((unsigned long long)sort_key(f[e]) << 32) | (uint32_t)~j;
        if (k < last && k > best) best = k;
      }
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
    if (tid == 0) {
      const int id = (int)~(uint32_t)best;
      ids[i] = id;
      lps[i] = (value(row.x[id]) - a.m) - ls;
    }
  }
}

// d logits of one row; g_logp and g_entropy may be null (no gradient).
template <typename T>
__global__ __launch_bounds__(256) void logprobs_bwd_kernel(const T* __restrict__ logits, long ld,
                                                           const int64_t* __restrict__ tokens,
                                                           const float* __restrict__ stat,
                                                           const float* __restrict__ g_logp, long gl_stride,
                                                           const float* __restrict__ g_entropy, long ge_stride,
                                                           T* __restrict__ dlogits, int V, long ignore_index) {
  constexpr int E = Row<T>::E;
  const long r = blockIdx.x;
  // chunks at the gradient's alignment (its rows are dense); the logits' may differ
  const Row<T> out(dlogits + r * (long)V, V);
  const T* x = logits + r * ld;
  const bool same = (uintptr_t)x % 16 == (uintptr_t)out.x % 16;
  const long tok = tokens[r];
  const float m = stat[3 * r], ls = stat[3 * r + 1], ent = stat[3 * r + 2];
  const float gl = !g_logp || tok == ignore_index ? 0.f
                   : tok >= 0 && tok < V          ? g_logp[r * gl_stride]
                                                  : __builtin_nanf("");
  const float ge = g_entropy ? g_entropy[r * ge_stride] : 0.f;
  for (int c = threadIdx.x; c < out.chunks; c += 256) {
    const int j0 = E * c - out.skip;
    const bool whole = j0 >= 0 && j0 + E <= V;
    float f[E], d[E];
    if (whole && same) {
      const uint4 u = __builtin_bit_cast(uint4, *reinterpret_cast<const f32x4*>(x + j0));
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (E == 8) {
          f[2 * e] = __uint_as_float(w[e] << 16);
          f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        } else {
          f[e] = __uint_as_float(w[e]);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = j0 + e >= 0 && j0 + e < V ? value(x[j0 + e]) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float lp = (f[e] - m) - ls, p = expf(lp);
      // 0 log 0 = 0 (the comparison keeps NaN)
      d[e] = (j0 + e == tok ? gl : 0.f) - p * fmaf(ge, (lp < -1e30f ? -1e30f : lp) + ent, gl);
    }
    if (whole) {
      if constexpr (E == 8) {
        bf16x8 o;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = (__bf16)d[e];
        __builtin_nontemporal_store(__builtin_bit_cast(f32x4, o), reinterpret_cast<f32x4*>(dlogits + r * (long)V + j0));
      } else {
        f32x4 o;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = d[e];
        __builtin_nontemporal_store(o, reinterpret_cast<f32x4*>(dlogits + r * (long)V + j0));
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (j0 + e >= 0 && j0 + e < V) {
          if constexpr (E == 8)
            dlogits[r * (long)V + j0 + e] = f32_to_bf16(d[e]);
          else
            dlogits[r * (long)V + j0 + e] = d[e];
        }
    }
  }
}

hipError_t launch_logprobs_fwd(const void* logits, bool bf16, long ld, const int64_t* tokens, float* logp,
                               float* entropy, float* stat, int64_t* top_ids, float* top_logp, long N, int V, int top,
                               long ignore_index, hipStream_t st) {
  auto run = [&](auto kernel, auto* x, int threads) {
    NAYLIS_TIMED("logprobs_fwd", st,
                 hipLaunchKernelGGL(kernel, dim3((unsigned)N), dim3(threads), 0, st, x, ld, tokens, logp, entropy,
                                    stat, top_ids, top_logp, V, top, ignore_index));
  };
  if (bf16)
    run(logprobs_fwd_kernel<bf16_t, 512>, (const bf16_t*)logits, 512);
  else
    run(logprobs_fwd_kernel<float, 512>, (const float*)logits, 512);
  return hipGetLastError();
}

hipError_t launch_logprobs_bwd(const void* logits, bool bf16, long ld, const int64_t* tokens, const float* stat,
                               const float* g_logp, long gl_stride, const float* g_entropy, long ge_stride,
                               void* dlogits, long N, int V, long ignore_index, hipStream_t st) {
  auto run = [&](auto kernel, auto* x) {
    typedef std::remove_const_t<std::remove_pointer_t<decltype(x)>> T;
    NAYLIS_TIMED("logprobs_bwd", st,
                 hipLaunchKernelGGL(kernel, dim3((unsigned)N), dim3(256), 0, st, x, ld, tokens, stat, g_logp,
                                    gl_stride, g_entropy, ge_stride, (T*)dlogits, V, ignore_index));
  };
  if (bf16)
    run(logprobs_bwd_kernel<bf16_t>, (const bf16_t*)logits);
  else
    run(logprobs_bwd_kernel<float>, (const float*)logits);
  return hipGetLastError();
}

}  // namespace naylis
