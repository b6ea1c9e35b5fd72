// Key / value cache in pages, and the attention of one new token over it.
//
// Pages (P, Hkv, page, hd) hold `page` consecutive tokens of one sequence, a
// head's rows together; table (B, W) names each sequence's pages in order.
// Rows are bf16, or e4m3 codes with one fp32 scale per row (the bank's form:
// scale = max|row| / 448, 1 for a row of zeros; code = e4m3(x / scale)).
//
// Attention: o[b, h] = softmax_n(scale q[b, h] . k[n]) v[n] over the sequence's
// tokens n < lens[b].  Bound by memory: every live K and V byte is read once
// (from L2 again when more than 16 query heads share a key head).
//
// Work is dealt in steps of 32 (bf16) or 64 (e4m3) tokens: each key head's
// steps of all sequences form one list, cut into equal ranges for its waves,
// so a long sequence among short ones keeps no wave waiting.  A wave that holds
// a whole sequence writes its result; the others leave (max, sum, o) partials
// that a second kernel joins.  Lengths stay on the device: each wave finds its
// range's first sequence by a scan over them.
//
// Per step a wave forms S^T = K Q^T (v_mfma_f32_16x16x32_bf16: 16 tokens x up
// to 16 query heads of the key head, zeros for missing ones) with K straight
// from memory, and O^T += V^T P^T with V through the wave's own piece of LDS,
// which transposes it; P leaves the accumulators as the B operand.  The next
// step's K and V are in flight meanwhile, and no barrier is needed.
#include "common.h"
#include "launch.h"
#include "packed_tiles.h"
#include "timing.h"

#include <algorithm>

namespace naylis {

namespace {

constexpr int kRowsMfma = 16;  // query heads of a product

__device__ __forceinline__ f32x4 mfma16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

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

// The wave's own LDS writes before its reads, and the other way round: LDS
// serves one wave's accesses in order, so only the compiler has to keep it.
__device__ __forceinline__ void lds_order() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
}

// Whether a table entry is a page.
__device__ __forceinline__ bool page_ok(int id, int pages) { return id >= 0 && id < pages; }

}  // namespace

// New rows into the cache, HD / 8 lanes a row.  Token t goes to sequence
// rows[t] (t itself without rows) at positions[t]; a position or a page outside
// the table or the cache (padding) writes nothing.
template <int HD, bool FP8>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedCacheDims c, const bf16_t* __restrict__ k,
                                                           const bf16_t* __restrict__ v,
                                                           const int32_t* __restrict__ table,
                                                           const int32_t* __restrict__ positions,
                                                           const int32_t* __restrict__ rows, PagedNew src) {
  constexpr int LANES = HD / 8;
  const long id = ((long)blockIdx.x * 256 + threadIdx.x) / LANES;  // (token, key head, K or V)
  const int piece = threadIdx.x % LANES;
  const bool is_v = id & 1;
  const long th = id >> 1, t = th / c.Hkv;
  const int h = (int)(th % c.Hkv);
  if (t >= src.T) return;
  const int b = rows ? rows[t] : (int)t, pos = positions[t];
  if (b < 0 || b >= c.B || pos < 0 || pos / c.page >= c.W) return;
  const int pg = table[(long)b * c.W + pos / c.page];
  if (!page_ok(pg, c.P)) return;
  const bf16_t* x = is_v ? v + t * src.ldv + h * src.hsv : k + t * src.ldk + h * src.hsk;
  const uint4 u = *reinterpret_cast<const uint4*>(x + 8 * piece);
  const long row = ((long)pg * c.Hkv + h) * c.page + pos % c.page;
  if constexpr (!FP8) {
    reinterpret_cast<uint4*>(is_v ? c.v : c.k)[row * LANES + piece] = u;
  } else {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    float f[8], top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      top = fmaxf(top, fmaxf(fabsf(f[2 * i]), fabsf(f[2 * i + 1])));
    }
    // the row's lanes are all here: they share t and so every return above
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
    if (piece == 0) (is_v ? c.v_scale : c.k_scale)[row] = s;
  }
}

namespace {

// Steps of the sequences before b, of all of them, and the steps of a wave's range.
template <int TOK>
struct StepList {
  const int32_t* lens;
  int B, cap;  // sequences, tokens that a table row holds

  __device__ __forceinline__ int len(int b) const { return b < B ? min(max(lens[b], 0), cap) : 0; }
  __device__ __forceinline__ int steps(int b) const { return (len(b) + TOK - 1) / TOK; }

  // sum of steps over sequences [0, b)
  __device__ __forceinline__ int before(int b) const {
    const int lane = threadIdx.x & 63;
    int t = 0;
    for (int i = lane; i < b; i += 64) t += steps(i);
    return __builtin_amdgcn_readfirstlane(wave_allsum_i32(t));
  }

  // the sequence that holds step `at` (at < before(B)) and its first step
  __device__ __forceinline__ void find(int at, int& b, int& first) const {
    const int lane = threadIdx.x & 63;
    int done = 0;
    for (int base = 0; base < B; base += 64) {
      const int here = steps(base + lane);
      int sum = here;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(sum, o, 64);
        if (lane >= o) sum += t;
      }
      const unsigned long long past = __ballot(done + sum > at);
      if (past) {
        const int src = __ffsll(past) - 1;
        b = base + src;
        first = done + __builtin_amdgcn_readlane(sum - here, src);
        return;
      }
      done += __builtin_amdgcn_readlane(sum, 63);
    }
    b = B;
    first = done;
  }
};

}  // namespace

// partials of (key head slice, wave, 0: the range's first sequence / 1: its last)
template <int HD>
__device__ __forceinline__ long part_row(const PagedSplit& p, int slice, int w, int slot) {
  return (((long)slice * p.waves + w) * 2 + slot) * p.rows;
}

// grid (waves / 4, slices): slice = (key head, 16 of its query heads)
template <int HD, bool FP8>
__global__ __launch_bounds__(256, 2) void paged_attn_kernel(PagedCacheDims c, const bf16_t* __restrict__ q, long ldq,
                                                            long hsq, const int32_t* __restrict__ table,
                                                            const int32_t* __restrict__ lens,
                                                            bf16_t* __restrict__ out, float* __restrict__ part,
                                                            float2* __restrict__ stat, PagedSplit p, float sc) {
  constexpr int TOK = FP8 ? 64 : 32;     // tokens of a step
  constexpr int NS = TOK / 16;           // its 16-token products
  constexpr int KS = HD / 32;            // products along the features
  constexpr int NT = HD / 16;            // 16-feature tiles of the output
  constexpr int RB = FP8 ? HD : 2 * HD;  // bytes of a cache row
  constexpr int KL = RB / 64;            // 16-byte loads of a lane for 16 tokens of K
  constexpr int VR = 1024 / RB;          // rows of V that a load of 64 lanes covers
  constexpr int VL = TOK / VR;           // such loads
  __shared__ __align__(16) uint8_t vt_all[4][TOK * 2 * HD];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint8_t* vt = vt_all[wave];
  const int w = blockIdx.x * 4 + wave, slice = blockIdx.y;
  const int kvh = slice / p.head_tiles, h0 = kRowsMfma * (slice % p.head_tiles);
  const int nh = min(kRowsMfma, c.G - h0);  // live query heads of the slice
  const StepList<TOK> list{lens, c.B, c.W * c.page};

  const int total = list.before(c.B);
  const int range = max((total + p.waves - 1) / p.waves, 1);
  int at = w * range;
  const int end = min(at + range, total);
  if (at >= end) return;
  int b, first;
  list.find(at, b, first);

  const long page_bytes = (long)c.Hkv * c.page * RB;
  const long head_off = (long)kvh * c.page * RB;
  const int shift = 31 - __clz(c.page);
  const int voff = lane * 16;                     // V: row lane / (RB / 16), piece lane % (RB / 16)
  const int koff = r16 * RB + g * 16;             // K: row r16, pieces g, g + 4, ..
  const int vrow = lane / (RB / 16), vpc = lane % (RB / 16);

  while (at < end && b < c.B) {
    const int n = list.len(b), nsteps = (n + TOK - 1) / TOK;
    const int s0 = at - first, s1 = min(end - first, nsteps);  // this wave's steps of sequence b
    bool bad = lens[b] > list.cap;                             // longer than its table

    bf16x8 qf[KS];
    {
      const bf16_t* qp = q + (long)b * ldq + (long)(kvh * c.G + h0 + min(r16, nh - 1)) * hsq;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        // feature order of the products: as the lane's 16-byte pieces of K hold them
        const int f = FP8 ? 64 * (ks >> 1) + 16 * g + 8 * (ks & 1) : 32 * ks + 8 * g;
        qf[ks] = *reinterpret_cast<const bf16x8*>(qp + f);
        if (r16 >= nh) qf[ks] = bf16x8{};
      }
    }
    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f32x4{};
    float m = kNegBig, l = 0.f;

    // pages of the next 64 products' tokens, one a lane
    int ids = 0, ids_at = -64;
    uint4 kx[NS][KL], vx[VL];
    float ksc[NS], vsc[NS];  // scales of token 16 i + r16
    auto load = [&](int step) {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const int t16 = step * NS + i;  // 16-token group of the sequence
        if (t16 >= ids_at + 64) {
          ids_at = t16;
          const int tok = (t16 + lane) << 4;
          ids = tok < n ? table[(long)b * c.W + (tok >> shift)] : 0;
        }
        int id = __builtin_amdgcn_readlane(ids, t16 - ids_at);
        if (!page_ok(id, c.P)) {
          bad = true;
          id = 0;
        }
        const int off = (t16 << 4) & (c.page - 1);
        const uint8_t* kp = (const uint8_t*)c.k + id * page_bytes + head_off + (long)off * RB;
        const uint8_t* vp = (const uint8_t*)c.v + id * page_bytes + head_off + (long)off * RB;
#pragma unroll
        for (int j = 0; j < KL; ++j) kx[i][j] = *reinterpret_cast<const uint4*>(kp + koff + 64 * j);
#pragma unroll
        for (int j = 0; j < VL / NS; ++j)
          vx[i * (VL / NS) + j] = *reinterpret_cast<const uint4*>(vp + voff + 1024 * j);
        if constexpr (FP8) {
          const long srow = ((long)id * c.Hkv + kvh) * c.page + off + r16;
          ksc[i] = c.k_scale[srow];
          vsc[i] = c.v_scale[srow];
        }
      }
    };
    load(s0);
    for (int s = s0; s < s1; ++s) {
      const int tok0 = s * TOK;
      // K fragments, then S^T: lane = query head r16, registers = tokens 16 i + 4 g + v
      f32x4 x[NS];
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        x[i] = f32x4{};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          bf16x8 kf;
          if constexpr (FP8) {
            const uint4 u = kx[i][ks >> 1];
            kf = (ks & 1) ? widen8(u.z, u.w) : widen8(u.x, u.y);
          } else {
            kf = __builtin_bit_cast(bf16x8, kx[i][ks]);
          }
          x[i] = mfma16(kf, qf[ks], x[i]);
        }
      }
      const bool tail = tok0 + TOK > n;
      // V rows to LDS as bf16; rows past the sequence as zeros, whatever the page holds there
#pragma unroll
      for (int j = 0; j < VL; ++j) {
        const int row = j * VR + vrow;
        uint4 u = vx[j];
        if (tail && tok0 + row >= n) u = make_uint4(0, 0, 0, 0);
        if constexpr (FP8) {
          const int ch = 2 * vpc;
          const int fx = HD == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3);
          *reinterpret_cast<bf16x8*>(vt + row * 2 * HD + ((ch ^ fx) << 4)) = widen8(u.x, u.y);
          *reinterpret_cast<bf16x8*>(vt + row * 2 * HD + (((ch + 1) ^ fx) << 4)) = widen8(u.z, u.w);
        } else {
          const int fx = HD == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3);
          *reinterpret_cast<uint4*>(vt + row * 2 * HD + ((vpc ^ fx) << 4)) = u;
        }
      }
      float kss[NS][4], vss[NS][4];
      if constexpr (FP8) {
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            kss[i][v] = __shfl(ksc[i], 4 * g + v, 64);
            vss[i][v] = __shfl(vsc[i], 4 * g + v, 64);
          }
      }
      lds_order();
      if (s + 1 < s1) load(s + 1);
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          if constexpr (FP8) x[i][v] *= kss[i][v];
          x[i][v] *= sc;
          if (tail && tok0 + 16 * i + 4 * g + v >= n) {
            x[i][v] = -INFINITY;
            if constexpr (FP8) vss[i][v] = 0.f;
          }
          mx = fmaxf(mx, x[i][v]);
        }
      const auto fmx = [](float a, float b) { return fmaxf(a, b); };
      mx = xor32_f32(xor16_f32(mx, fmx), fmx);
      const float mn = fmaxf(m, mx), al = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= al;
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t] *= al;
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          x[i][v] = __builtin_amdgcn_exp2f(x[i][v] - mn);
          l += x[i][v];
          if constexpr (FP8) x[i][v] *= vss[i][v];
        }
      // O^T += V^T P^T over 32 tokens: registers of two products are the B operand
#pragma unroll
      for (int i = 0; i < NS; i += 2) {
        bf16x8 pf;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pf[e] = (__bf16)x[i][e];
          pf[4 + e] = (__bf16)x[i + 1][e];
        }
        const int rlo = 16 * i + 4 * g + (r16 >> 2), rhi = rlo + 16;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int ch = 2 * t + ((r16 & 3) >> 1), b8 = 8 * (r16 & 1);
          const int flo = HD == 128 ? 2 * (rlo & 7) : 2 * ((rlo >> 1) & 3);
          const int fhi = HD == 128 ? 2 * (rhi & 7) : 2 * ((rhi >> 1) & 3);
          const v4i16 lo = lds_read_tr16(reinterpret_cast<const bf16_t*>(vt + rlo * 2 * HD + ((ch ^ flo) << 4) + b8));
          const v4i16 hi = lds_read_tr16(reinterpret_cast<const bf16_t*>(vt + rhi * 2 * HD + ((ch ^ fhi) << 4) + b8));
          typedef short v8i16 __attribute__((ext_vector_type(8)));
          const v8i16 vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
          acc[t] = mfma16(__builtin_bit_cast(bf16x8, vf), pf, acc[t]);
        }
      }
      lds_order();
    }
    const auto add = [](float a, float b2) { return a + b2; };
    l = xor32_f32(xor16_f32(l, add), add);
    if (bad) l = __builtin_nanf("");  // a page that is none: the sequence's result is NaN
    if (r16 < nh) {
      const int h = kvh * c.G + h0 + r16;
      if (s0 == 0 && s1 == nsteps) {
        const float inv = 1.f / l;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          bf16x4 o;
#pragma unroll
          for (int v = 0; v < 4; ++v) o[v] = (__bf16)(acc[t][v] * inv);
          *reinterpret_cast<bf16x4*>(out + ((long)b * c.Hkv * c.G + h) * HD + 16 * t + 4 * g) = o;
        }
      } else {
        const long row = part_row<HD>(p, slice, w, at == w * range ? 0 : 1) + r16;
#pragma unroll
        for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4*>(part + row * HD + 16 * t + 4 * g) = acc[t];
        if (g == 0) stat[row] = make_float2(m, l);
      }
    }
    at = first + s1;
    first += nsteps;
    ++b;
    while (b < c.B && list.steps(b) == 0) ++b;  // sequences without tokens hold no step
  }
}

// Joins a sequence's partials, or writes zeros for a sequence without tokens;
// nothing where one wave held it whole.  Grid (H, B), HD threads a range of waves.
template <int HD, int TOK>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedCacheDims c, const int32_t* __restrict__ lens,
                                                         bf16_t* __restrict__ out, const float* __restrict__ part,
                                                         const float2* __restrict__ stat, PagedSplit p) {
  constexpr int NG = 256 / HD;  // groups of threads, each over every NG-th wave's partial
  __shared__ float red[NG][HD];
  __shared__ float2 reds[NG];
  const int h = blockIdx.x, b = blockIdx.y, f = threadIdx.x % HD, gi = threadIdx.x / HD;
  const StepList<TOK> list{lens, c.B, c.W * c.page};
  const int n = list.steps(b);
  bf16_t* o = out + ((long)b * c.Hkv * c.G + h) * HD;
  if (n == 0) {
    if (gi == 0) o[f] = 0;
    return;
  }
  const int total = list.before(c.B), range = max((total + p.waves - 1) / p.waves, 1);
  const int first = list.before(b), w0 = first / range, w1 = (first + n - 1) / range;
  if (w0 == w1) return;
  const int kvh = h / c.G, hr = h % c.G, slice = kvh * p.head_tiles + hr / kRowsMfma;
  float m = kNegBig, l = 0.f, a = 0.f;
  for (int w = w0 + gi; w <= w1; w += NG) {
    // the wave's first sequence, unless its range begins before this one
    const long row = part_row<HD>(p, slice, w, w * range >= first ? 0 : 1) + hr % kRowsMfma;
    const float2 st = stat[row];
    const float mn = fmaxf(m, st.x), x = __builtin_amdgcn_exp2f(m - mn), y = __builtin_amdgcn_exp2f(st.x - mn);
    a = a * x + part[row * HD + f] * y;
    l = l * x + st.y * y;
    m = mn;
  }
  red[gi][f] = a;
  if (f == 0) reds[gi] = make_float2(m, l);
  __syncthreads();
  if (gi) return;
  float mn = kNegBig;
#pragma unroll
  for (int i = 0; i < NG; ++i) mn = fmaxf(mn, reds[i].x);
  a = l = 0.f;
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const float y = __builtin_amdgcn_exp2f(reds[i].x - mn);
    a += red[i][f] * y;
    l += reds[i].y * y;
  }
  o[f] = f32_to_bf16(a / l);
}

// Waves for each slice: 8 a CU over all slices, a whole number of workgroups,
// and no more than the tables' steps (rounded up).
PagedSplit paged_split(const PagedCacheDims& c, int hd, bool fp8) {
  PagedSplit p;
  p.head_tiles = (c.G + kRowsMfma - 1) / kRowsMfma;
  p.rows = std::min(c.G, kRowsMfma);
  const long slices = (long)c.Hkv * p.head_tiles;
  const int tok = fp8 ? 64 : 32;
  const long cap = (long)c.B * (((long)c.W * c.page + tok - 1) / tok);
  const long waves = std::min(std::max(2048 / slices, 4L), std::max(cap, 1L));
  p.waves = (int)((waves + 3) / 4 * 4);
  return p;
}

size_t paged_part_floats(const PagedCacheDims& c, const PagedSplit& p, int hd) {
  return (size_t)c.Hkv * p.head_tiles * p.waves * 2 * p.rows * hd;
}

size_t paged_ws_bytes(const PagedCacheDims& c, int hd, bool fp8) {
  const PagedSplit p = paged_split(c, hd, fp8);
  return paged_part_floats(c, p, hd) * 4 + (size_t)c.Hkv * p.head_tiles * p.waves * 2 * p.rows * 8;
}

hipError_t launch_paged_append(const PagedCacheDims& c, int hd, bool fp8, const void* k, const void* v,
                               const int32_t* table, const int32_t* positions, const int32_t* rows,
                               const PagedNew& src, hipStream_t st) {
  const long threads = src.T * c.Hkv * 2 * (hd / 8);
  auto run = [&](auto kernel) {
    NAYLIS_TIMED("paged_append", st,
                 hipLaunchKernelGGL(kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, c,
                                    (const bf16_t*)k, (const bf16_t*)v, table, positions, rows, src));
  };
  if (hd == 64)
    fp8 ? run(paged_append_kernel<64, true>) : run(paged_append_kernel<64, false>);
  else
    fp8 ? run(paged_append_kernel<128, true>) : run(paged_append_kernel<128, false>);
  return hipGetLastError();
}

hipError_t launch_paged_attn(const PagedCacheDims& c, int hd, bool fp8, const void* q, long ldq, long hsq,
                             const int32_t* table, const int32_t* lens, void* out, void* ws, float scale,
                             hipStream_t st) {
  const PagedSplit p = paged_split(c, hd, fp8);
  float* part = (float*)ws;
  float2* stat = (float2*)(part + paged_part_floats(c, p, hd));
  auto run = [&](auto kernel) {
    NAYLIS_TIMED("paged_attn", st,
                 hipLaunchKernelGGL(kernel, dim3(p.waves / 4, c.Hkv * p.head_tiles), dim3(256), 0, st, c,
                                    (const bf16_t*)q, ldq, hsq, table, lens, (bf16_t*)out, part, stat, p,
                                    scale * kLog2e));
  };
  if (hd == 64)
    fp8 ? run(paged_attn_kernel<64, true>) : run(paged_attn_kernel<64, false>);
  else
    fp8 ? run(paged_attn_kernel<128, true>) : run(paged_attn_kernel<128, false>);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  auto join = [&](auto kernel) {
    NAYLIS_TIMED("paged_join", st,
                 hipLaunchKernelGGL(kernel, dim3(c.Hkv * c.G, c.B), dim3(256), 0, st, c, lens, (bf16_t*)out,
                                    (const float*)part, (const float2*)stat, p));
  };
  if (hd == 64)
    fp8 ? join(paged_join_kernel<64, 64>) : join(paged_join_kernel<64, 32>);
  else
    fp8 ? join(paged_join_kernel<128, 64>) : join(paged_join_kernel<128, 32>);
  return hipGetLastError();
}

}  // namespace naylis
