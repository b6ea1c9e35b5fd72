// Device code shared by the kernels that read and write the paged cache.
#pragma once
#include <type_traits>

#include "common.h"
#include "launch.h"

namespace naylis {

// eight e4m3 codes as bf16 (exact)
__device__ __forceinline__ bf16x8 widen8(uint32_t lo, uint32_t hi) {
  bf16x8 r;
  const uint32_t w[2] = {lo, hi};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
    const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
    r[4 * i] = (__bf16)a[0];
    r[4 * i + 1] = (__bf16)a[1];
    r[4 * i + 2] = (__bf16)b[0];
    r[4 * i + 3] = (__bf16)b[1];
  }
  return r;
}

// eight e2m1 codes, the first in the low bits, times 2^(e - 127) as bf16: exact, NaN for e = 255.
// The conversion reads nothing of the scale but its exponent, and takes 0 there for 2^-127.
__device__ __forceinline__ bf16x8 widen8_e2m1(uint32_t codes, uint32_t e) {
  const float s = __uint_as_float(e << 23);
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 0);
  const auto b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 1);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 2);
  const auto d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Whether a table entry is a page.
__device__ __forceinline__ bool page_ok(int id, int pages) { return id >= 0 && id < pages; }

// Eight features of a cache row, 8 * piece .., as codes.  The row's HD / 8 lanes
// are neighbours and call together: they share its scale (e4m3: max|row| / 448 in
// fp32, 1 for a row of zeros) or fours of them a block's (e2m1: 2^(floor(log2
// max|block|) - 2), at least 2^-126, so the largest value falls on 4 .. 8 of codes
// that end at 6; a block with an infinity or a NaN is NaN).
template <int HD, PagedFormat FMT>
__device__ __forceinline__ void store_codes(const PagedCacheDims& c, bool is_v, long row, int piece,
                                            const float (&f)[8]) {
  constexpr int LANES = HD / 8;
  if constexpr (FMT == kPagedE4m3) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(f[2 * i]), fabsf(f[2 * i + 1])));
    const auto mx = [](float a, float b) { return fmaxf(a, b); };
    top = mx(top, dpp_f32<0xb1>(top));
    top = mx(top, dpp_f32<0x4e>(top));
    top = mx(top, dpp_f32<0x141>(top));
    if constexpr (LANES == 16) top = mx(top, dpp_f32<0x140>(top));
    const float s = top > 0.f ? top / 448.f : 1.f;
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0] / s, f[1] / s, lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[2] / s, f[3] / s, lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4] / s, f[5] / s, hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[6] / s, f[7] / s, hi, true);
    reinterpret_cast<uint2*>(is_v ? c.v : c.k)[row * LANES + piece] = make_uint2((uint32_t)lo, (uint32_t)hi);
    if (piece == 0) reinterpret_cast<float*>(is_v ? c.v_scale : c.k_scale)[row] = s;
  } else {
    static_assert(FMT == kPagedE2m1, "codes are e4m3 or e2m1");
    int top = 0;  // of the bits: NaN above infinity above all numbers
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_int(f[i]) & 0x7fffffff);
    top = max(top, dpp_i32<0xb1>(top));
    top = max(top, dpp_i32<0x4e>(top));
    const int e = top >> 23, byte = e == 255 ? 255 : max(e - 2, 1);
    const float s = __uint_as_float((uint32_t)byte << 23);
    uint32_t codes = 0;  // rounded to nearest even, at most 6
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[0], f[1], s, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[2], f[3], s, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[4], f[5], s, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[6], f[7], s, 3);
    reinterpret_cast<uint32_t*>(is_v ? c.v : c.k)[row * LANES + piece] = codes;
    if (piece % 4 == 0)
      reinterpret_cast<uint8_t*>(is_v ? c.v_scale : c.k_scale)[row * (HD / 32) + piece / 4] = (uint8_t)byte;
  }
}

template <PagedFormat F>
using Format = std::integral_constant<PagedFormat, F>;

// f(head dim, format) as compile-time constants
template <typename F>
void with_format(int hd, PagedFormat fmt, F f) {
  auto go = [&](auto d) {
    if (fmt == kPagedBf16)
      f(d, Format<kPagedBf16>{});
    else if (fmt == kPagedE4m3)
      f(d, Format<kPagedE4m3>{});
    else
      f(d, Format<kPagedE2m1>{});
  };
  hd == 64 ? go(std::integral_constant<int, 64>{}) : go(std::integral_constant<int, 128>{});
}

}  // namespace naylis
