// New tokens rotated to their positions and into the paged cache, and the
// cache's sequences back as dense rows.
//
// Rotation: of the first 2 half features of a row, pair (x_i, x_{i + half}) turns
// by the angle position * inv_freq[i]:
//   y_i = x_i cos - x_{i + half} sin,  y_{i + half} = x_{i + half} cos + x_i sin.
// Angles, their reduction and cos / sin are fp64 (far positions lose their angle
// in fp32: at 131072 the last bit is 2^-7), cos and sin then fp32, times the
// scaling; products and sum are rounded in fp32 each, the result once to the
// cache's type.  A workgroup takes a token: its angles once, then all its rows.
// Bound by memory: 8191 tokens of 32 + 2 x 8 heads of 128 into bf16 pages, 201 MB, 41 us
// (4.9 TB/s, a large copy's rate); 256 tokens into e4m3 pages 4.3 us, two of which are
// angle, page and row one after another.
//
// Back: a lane widens 8 features.  16381 tokens, 16 heads of 64, from e4m3 pages: 18 us
// for 103 MB (5.6 TB/s, two thirds of it written); bf16 pages 23.6 for 134 MB.
#include "common.h"
#include "launch.h"
#include "paged_common.h"
#include "timing.h"

#include <algorithm>

namespace naylis {

namespace {

constexpr int kChunkThreads = 256;

// sin and cos of x: x less a multiple of pi / 2 in two parts (Cody and Waite), then
// the Taylor series up to r^17 / r^16 on |r| <= pi / 4: what they leave out is 8e-20
// and 2e-18, fp64's roundings some 1e-16.
__device__ __forceinline__ void sincos64(double x, float& sine, float& cosine) {
  const double n = rint(x * 0.63661977236758134308);
  double r = __builtin_fma(-n, 1.57079632679489661923, x);
  r = __builtin_fma(-n, 6.123233995736766036e-17, r);
  const double z = r * r;
  double s = 1.0 / 355687428096000.0;  // 1 / 17!
  s = __builtin_fma(s, z, -1.0 / 1307674368000.0);
  s = __builtin_fma(s, z, 1.0 / 6227020800.0);
  s = __builtin_fma(s, z, -1.0 / 39916800.0);
  s = __builtin_fma(s, z, 1.0 / 362880.0);
  s = __builtin_fma(s, z, -1.0 / 5040.0);
  s = __builtin_fma(s, z, 1.0 / 120.0);
  s = __builtin_fma(s, z, -1.0 / 6.0);
  s = __builtin_fma(s * z, r, r);
  double c = 1.0 / 20922789888000.0;  // 1 / 16!
  c = __builtin_fma(c, z, -1.0 / 87178291200.0);
  c = __builtin_fma(c, z, 1.0 / 479001600.0);
  c = __builtin_fma(c, z, -1.0 / 3628800.0);
  c = __builtin_fma(c, z, 1.0 / 40320.0);
  c = __builtin_fma(c, z, -1.0 / 720.0);
  c = __builtin_fma(c, z, 1.0 / 24.0);
  c = __builtin_fma(c, z, -0.5);
  c = __builtin_fma(c, z, 1.0);
  const int q = (int)(n - 4.0 * rint(n * 0.25));  // n mod 4 in -2 .. 2
  const double a = q & 1 ? c : s, b = q & 1 ? s : c;
  sine = (float)(q & 2 ? -a : a);
  cosine = (float)((q + 1) & 2 ? -b : b);
}

__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ uint4 round8(const float (&f)[8]) {
  bf16x8 o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = (__bf16)f[e];
  return __builtin_bit_cast(uint4, o);
}

}  // namespace

// Grid (T, shares of a token's rows): rows of q, k and v of token t, HD / 8 lanes
// each; k and v go to token positions[t] of sequence rows[t] (t itself without
// rows), or nowhere where that lies outside the table or the cache.
template <int HD, PagedFormat FMT>
__global__ __launch_bounds__(kChunkThreads) void paged_rope_kernel(PagedCacheDims c, PagedRope r,
                                                                   const int32_t* __restrict__ table,
                                                                   const int32_t* __restrict__ positions,
                                                                   const int32_t* __restrict__ rows) {
  constexpr int LANES = HD / 8, RPW = kChunkThreads / LANES;  // lanes of a row, rows at a time
  __shared__ float2 turn[HD / 2];  // (cos, sin)
  const long t = blockIdx.x;
  const int tid = threadIdx.x, piece = tid % LANES, pos = positions[t];
  if (tid < r.half) {
    float s, co;
    sincos64((double)pos * (double)r.inv_freq[tid], s, co);
    turn[tid] = make_float2(mul_rn(co, r.scaling), mul_rn(s, r.scaling));
  }
  const int b = rows ? rows[t] : (int)t;
  long place = -1;  // the cache row of head 0
  if (b >= 0 && b < c.B && pos >= 0 && pos / c.page < c.W) {
    const int pg = table[(long)b * c.W + pos / c.page];
    if (page_ok(pg, c.P)) place = (long)pg * c.Hkv * c.page + pos % c.page;
  }
  __syncthreads();
  const int half8 = r.half / 8;
  const bool turned = piece < 2 * half8, low = piece < half8;
  const int other = low ? piece + half8 : piece - half8;
  float2 cs[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) cs[e] = turned ? turn[8 * (low ? piece : other) + e] : make_float2(1.f, 0.f);
  const int all = r.H + 2 * c.Hkv;
  for (int row = blockIdx.y * RPW + tid / LANES; row < all; row += gridDim.y * RPW) {
    const bool is_q = row < r.H, is_v = row >= r.H + c.Hkv;
    const int h = is_q ? row : is_v ? row - r.H - c.Hkv : row - r.H;
    if (!is_q && place < 0) continue;
    const bf16_t* x = is_q   ? (const bf16_t*)r.q + t * r.ldq + h * r.hsq
                      : is_v ? (const bf16_t*)r.v + t * r.ldv + h * r.hsv
                             : (const bf16_t*)r.k + t * r.ldk + h * r.hsk;
    uint4 u = *reinterpret_cast<const uint4*>(x + 8 * piece);
    float f[8];
    unpack8(u, f);
    if (turned && !is_v) {
      float g[8];
      unpack8(*reinterpret_cast<const uint4*>(x + 8 * other), g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = mul_rn(f[e], cs[e].x), o = mul_rn(g[e], cs[e].y);
        f[e] = low ? add_rn(a, -o) : add_rn(a, o);
      }
      u = round8(f);
    }
    if (is_q) {
      reinterpret_cast<uint4*>(r.q_out)[(t * r.H + h) * LANES + piece] = u;
    } else {
      const long at = place + (long)h * c.page;
      if constexpr (FMT == kPagedBf16)
        reinterpret_cast<uint4*>(is_v ? c.v : c.k)[at * LANES + piece] = u;
      else
        store_codes<HD, FMT>(c, is_v, at, piece, f);
    }
  }
}

// Rows t of k_out, v_out (T, Hkv, HD) are token t - cu[b] of the sequence b that
// holds them: 0 outside the sequences, NaN for a page outside the cache or a
// token past the table's row.  Grid (tiles of 16 tokens, shares of their rows).
constexpr int kGatherTokens = 16;
template <int HD, PagedFormat FMT>
__global__ __launch_bounds__(kChunkThreads) void paged_gather_kernel(PagedCacheDims c,
                                                                     const int32_t* __restrict__ table,
                                                                     const int32_t* __restrict__ cu,
                                                                     bf16_t* __restrict__ k_out,
                                                                     bf16_t* __restrict__ v_out, long T) {
  constexpr int LANES = HD / 8, RPW = kChunkThreads / LANES;
  __shared__ long places[kGatherTokens];  // cache row of head 0; -1: no sequence, -2: no page
  const int tid = threadIdx.x, piece = tid % LANES;
  const long t0 = (long)blockIdx.x * kGatherTokens;
  if (tid < kGatherTokens) {
    const long t = t0 + tid;
    long place = -1;
    if (t < T && t >= cu[0] && t < cu[c.B]) {
      int lo = 0, hi = c.B;  // cu[lo] <= t < cu[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        (cu[mid] <= t ? lo : hi) = mid;
      }
      const long pos = t - cu[lo];
      place = -2;
      if (pos >= 0 && pos / c.page < c.W) {
        const int pg = table[(long)lo * c.W + pos / c.page];
        if (page_ok(pg, c.P)) place = (long)pg * c.Hkv * c.page + pos % c.page;
      }
    }
    places[tid] = place;
  }
  __syncthreads();
  // a head's tokens are neighbours in a page: rows go token by token within a head
  const int all = 2 * c.Hkv * kGatherTokens;
#pragma unroll 4
  for (int row = blockIdx.y * RPW + tid / LANES; row < all; row += gridDim.y * RPW) {
    const int i = row % kGatherTokens, hv = row / kGatherTokens;
    const bool is_v = hv >= c.Hkv;
    const int h = is_v ? hv - c.Hkv : hv;
    if (t0 + i >= T) continue;
    const long place = places[i], at = place + (long)h * c.page;
    const void* pages = is_v ? c.v : c.k;
    const void* scales = is_v ? c.v_scale : c.k_scale;
    uint4 o = make_uint4(0, 0, 0, 0);
    if (place == -2) {
      o = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
    } else if (place >= 0) {
      if constexpr (FMT == kPagedBf16) {
        o = reinterpret_cast<const uint4*>(pages)[at * LANES + piece];
      } else if constexpr (FMT == kPagedE4m3) {
        const uint2 u = reinterpret_cast<const uint2*>(pages)[at * LANES + piece];
        const float s = reinterpret_cast<const float*>(scales)[at];
        float f[8];
        const bf16x8 x = widen8(u.x, u.y);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (float)x[e] * s;
        o = round8(f);
      } else {
        const uint32_t u = reinterpret_cast<const uint32_t*>(pages)[at * LANES + piece];
        const uint32_t e = reinterpret_cast<const uint8_t*>(scales)[at * (HD / 32) + piece / 4];
        o = __builtin_bit_cast(uint4, widen8_e2m1(u, e));
      }
    }
    reinterpret_cast<uint4*>(is_v ? v_out : k_out)[((t0 + i) * c.Hkv + h) * LANES + piece] = o;
  }
}

namespace {

// Workgroups that share the rows of one of n: as many as fill the chip.
unsigned shares(long n, int rows, int at_a_time) {
  const long passes = (rows + at_a_time - 1) / at_a_time;
  return (unsigned)std::min(passes, std::max(1l, 2048 / std::max(n, 1l)));
}

}  // namespace

hipError_t launch_paged_append_rope(const PagedCacheDims& c, int hd, PagedFormat fmt, const PagedRope& r,
                                    const int32_t* table, const int32_t* positions, const int32_t* rows,
                                    hipStream_t st) {
  const dim3 grid((unsigned)r.T, shares(r.T, r.H + 2 * c.Hkv, kChunkThreads / (hd / 8)));
  with_format(hd, fmt, [&](auto d, auto f) {
    NAYLIS_TIMED("paged_append_rope", st,
                 hipLaunchKernelGGL((paged_rope_kernel<decltype(d)::value, decltype(f)::value>), grid,
                                    dim3(kChunkThreads), 0, st, c, r, table, positions, rows));
  });
  return hipGetLastError();
}

hipError_t launch_paged_gather(const PagedCacheDims& c, int hd, PagedFormat fmt, const int32_t* table,
                               const int32_t* cu, void* k_out, void* v_out, long T, hipStream_t st) {
  const long tiles = (T + kGatherTokens - 1) / kGatherTokens;
  const dim3 grid((unsigned)tiles, shares(tiles, 2 * c.Hkv * kGatherTokens, kChunkThreads / (hd / 8)));
  with_format(hd, fmt, [&](auto d, auto f) {
    NAYLIS_TIMED("paged_gather", st,
                 hipLaunchKernelGGL((paged_gather_kernel<decltype(d)::value, decltype(f)::value>), grid,
                                    dim3(kChunkThreads), 0, st, c, table, cu, (bf16_t*)k_out, (bf16_t*)v_out, T));
  });
  return hipGetLastError();
}

}  // namespace naylis
