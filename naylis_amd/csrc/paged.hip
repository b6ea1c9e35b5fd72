// Key / value cache in pages, and the attention of one new token over it.
//
// Pages (P, Hkv, page, hd) hold `page` consecutive tokens of one sequence, a
// head's rows together; table (B, W) names each sequence's pages in order.
// Rows are bf16, or e4m3 codes with one fp32 scale per row (the bank's form:
// scale = max|row| / 448, 1 for a row of zeros; code = e4m3(x / scale)).
//
// Attention: o[b, h] = softmax_n(scale q[b, h] . k[n]) v[n] over the sequence's
// tokens n < lens[b].  Bound by memory: every live K and V byte is read once
// (again for each further 16 query heads of a key head), past the caches.
//
// Work is dealt in steps of 32 tokens: each slice's (key head's) steps of all
// sequences form one list, cut into equal ranges for its workgroups and those
// into four for their waves, so a long sequence among short ones keeps no
// wave waiting.  The waves of a workgroup join what they hold of one sequence
// in LDS, all of it read at once; what several workgroups hold of it goes to a
// second kernel as (max, sum, o) partials.  Lengths stay on the device: each wave
// finds its range's first sequence by two scans over them, and leaves each
// sequence's first step for the second kernel (4096 sequences of up to 1024 tokens,
// one key head of 64: 104 us and 25; with scans of 64 sequences a round 393 and 234).
//
// Per step a wave forms S^T = K Q^T (v_mfma_f32_16x16x32_bf16: 16 tokens x up
// to 16 query heads of the key head, zeros for missing ones) with K straight
// from memory, and O^T += V^T P^T with V through the wave's own piece of LDS,
// which transposes it; P leaves the accumulators as the B operand, rounded to
// bf16 (with e4m3 pages, times V's scale).  The next step's K is loaded as soon
// as the products have read this one's, V as soon as LDS has, and no barrier is
// needed.  Loads bypass the caches (a tenth of the time): 64 sequences of up to 4096
// tokens, 8 key heads of 128, 588 MB: 98 us (6.0 TB/s; 5 of them the join and its
// launch).  Three contexts of 65537 .. 131072 tokens, e4m3, 747 MB: 123 us (6.1 TB/s);
// in steps of 64 tokens 134 (256 registers).  One sequence of 500 tokens, 16 heads of
// 64: 7.0 us, a chain of dependent loads (length, page, rows) that fill nothing.
#include "common.h"
#include "launch.h"
#include "packed_tiles.h"
#include "timing.h"

#include <algorithm>
#include <type_traits>

namespace naylis {

namespace {

constexpr int kRowsMfma = 16;       // query heads of a product
constexpr int kPagedStep = 32;      // tokens of a step
constexpr int kPagedMaxWgs = 512;   // workgroups that share a slice's steps

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

// The list of all sequences' steps.  A lane looks after an equal chunk of the
// sequences, so that a place is found with one scan over the lanes and one over
// a chunk, whatever their number.
struct StepList {
  const int32_t* lens;
  int B, cap;  // sequences, tokens that a table row holds

  // (any b: loads of several at once are not held up by a comparison)
  __device__ __forceinline__ int len(int b) const {
    const int n = lens[min(b, B - 1)];
    return b < B ? min(max(n, 0), cap) : 0;
  }
  __device__ __forceinline__ int steps(int b) const { return (len(b) + kPagedStep - 1) / kPagedStep; }

  static __device__ __forceinline__ int inclusive(int x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int t = __shfl_up(x, o, 64);
      if (lane >= o) x += t;
    }
    return x;
  }

  __device__ __forceinline__ int chunk() const { return (B + 63) / 64; }
  // steps of the lane's chunk, and of all up to it
  __device__ __forceinline__ int2 chunks() const {
    const int n = chunk(), b = (threadIdx.x & 63) * n;
    int own = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) own += steps(b + i);
    return make_int2(own, inclusive(own));
  }

  // the sequence that holds step `at` (one of the list's) and its first step
  __device__ __forceinline__ void find(int at, const int2& sums, int& b, int& first) const {
    const int lane = threadIdx.x & 63, n = chunk();
    const int src = max(__ffsll((unsigned long long)__ballot(sums.y > at)) - 1, 0);
    b = src * n;
    first = __builtin_amdgcn_readlane(sums.y - sums.x, src);
    if (n == 1) return;
    for (int i = 0; i < n; i += 64) {
      const int own = i + lane < n ? steps(b + lane) : 0, sum = inclusive(own);
      const unsigned long long past = __ballot(first + sum > at);
      if (past) {
        const int in = __ffsll(past) - 1;
        b += in;
        first += __builtin_amdgcn_readlane(sum - own, in);
        return;
      }
      b += 64;
      first += __builtin_amdgcn_readlane(sum, 63);
    }
  }

  // the first sequence from b on that has tokens, or B
  __device__ __forceinline__ int next(int b) const {
    for (; b < B; b += 64) {
      const unsigned long long live = __ballot(len(b + (int)(threadIdx.x & 63)) > 0);
      if (live) return b + __ffsll(live) - 1;
    }
    return B;
  }
};

// What the waves of a workgroup hand each other: up to two partials each (the
// first and the last sequence of a wave's range), in order.
struct PartSeq {
  int b, first, steps;  // sequence (-1: none), its first step in the list, its steps
};

// LDS of a wave: its V tile (32 tokens), where its last partial goes too (16
// rows of fp32, once the tile is no longer needed), then its first partial.
template <int HD, int ROWS>
constexpr int kWaveLds = 32 * 2 * HD + ROWS * HD * 4;
template <int HD>
__device__ __forceinline__ int part_offset(int slot) {
  static_assert(kRowsMfma * 4 == 32 * 2, "a partial fits the V tile");
  return slot == 0 ? 32 * 2 * HD : 0;
}

template <int HD>
__device__ __forceinline__ int v_slot(int row, int chunk) {  // byte of a 16-byte chunk in the V tile
  const int f = HD == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3);
  return row * 2 * HD + ((chunk ^ f) << 4);
}

__device__ __forceinline__ uint4 load_once16(const uint8_t* p) {
  return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p)));
}

}  // namespace

// partials of (slice, workgroup, 0: the first sequence of its range / 1: the last)
__device__ __forceinline__ long part_row(const PagedSplit& p, int slice, int wg, int slot) {
  return (((long)slice * p.wgs + wg) * 2 + slot) * p.rows;
}

// grid (workgroups of a slice, slices): slice = (key head, 16 of its query heads).
// A workgroup takes a range of the step list, or (p.whole) the sequence of its
// number, its waves an equal share each.
// ROWS: partials' rows, at least the query heads of a slice.
template <int HD, bool FP8, int ROWS>
__global__ __launch_bounds__(256, 2) void paged_attn_kernel(PagedCacheDims c, const bf16_t* __restrict__ q, long ldq,
                                                            long hsq, const int32_t* __restrict__ table,
                                                            const int32_t* __restrict__ lens,
                                                            bf16_t* __restrict__ out, float* __restrict__ part,
                                                            float2* __restrict__ stat, int* __restrict__ starts,
                                                            PagedSplit p, float sc) {
  constexpr int TOK = kPagedStep;        // tokens of a step
  constexpr int NS = TOK / 16;           // its 16-token products
  constexpr int KS = HD / 32;            // products along the features
  constexpr int NT = HD / 16;            // 16-feature tiles of the output
  constexpr int RB = FP8 ? HD : 2 * HD;  // bytes of a cache row
  constexpr int KL = RB / 64;            // 16-byte loads of a lane for 16 tokens of K
  constexpr int VR = 1024 / RB;          // rows of V that a load of 64 lanes covers
  constexpr int VL = TOK / VR;           // such loads
  __shared__ __align__(16) uint8_t lds[4 * kWaveLds<HD, ROWS>];
  __shared__ PartSeq seqs[8];
  __shared__ float2 stats[8][ROWS];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint8_t* vt = lds + wave * kWaveLds<HD, ROWS>;
  const int wg = blockIdx.x, slice = blockIdx.y;
  const int kvh = slice / p.head_tiles, h0 = kRowsMfma * (slice % p.head_tiles);
  const int nh = min(kRowsMfma, c.G - h0);  // live query heads of the slice
  const int H = c.Hkv * c.G, hbase = kvh * c.G + h0;
  const StepList list{lens, c.B, c.W * c.page};

  int wg0, wg1, at, end, b = wg, first = 0;
  int2 sums = make_int2(0, 0);
  if (p.whole) {
    wg0 = 0;
    wg1 = list.steps(wg);
  } else {
    sums = list.chunks();
    const int total = __builtin_amdgcn_readlane(sums.y, 63), range = max((total + p.wgs - 1) / p.wgs, 1);
    if (tid == 0 && wg == 0 && slice == 0) starts[c.B] = total;
    wg0 = min(wg * range, total);
    wg1 = min(wg0 + range, total);
  }
  {
    const int share = (wg1 - wg0 + 3) / 4;
    at = min(wg0 + wave * share, wg1);
    end = min(at + share, wg1);
  }
  if (!p.whole && at < end) list.find(at, sums, b, first);
  if (lane < 2) seqs[2 * wave + lane].b = -1;

  const int shift = 31 - __clz(c.page);
  const int voff = lane * 16;          // V: row lane / (RB / 16), piece lane % (RB / 16)
  const int koff = r16 * RB + g * 16;  // K: row r16, pieces g, g + 4, ..
  const int vrow = lane / (RB / 16), vpc = lane % (RB / 16);
  const int begin = at;

  while (at < end && b < c.B) {
    const int n = list.len(b), nsteps = (n + TOK - 1) / TOK;
    const int s0 = at - first, s1 = min(end - first, nsteps);  // this wave's steps of sequence b
    bool bad = lens[b] > list.cap;                             // longer than its table
    if (!p.whole && s0 == 0 && slice == 0 && lane == 0) starts[b] = first;

    bf16x8 qf[KS];
    {
      const bf16_t* qp = q + (long)b * ldq + (long)(hbase + min(r16, nh - 1)) * hsq;
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
    float m = kLowest, l = 0.f;

    // pages of the next 64 products' tokens, one a lane
    int ids = 0, ids_at = -64;
    uint4 kx[NS][KL], vx[VL];
    f32x4 ksc[NS], vsc[NS];  // scales of tokens 16 i + 4 g ..
    long row16[NS];          // cache row of each 16-token group of the step being loaded
    auto find_pages = [&](int step) {
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
        row16[i] = ((long)id * c.Hkv + kvh) * c.page + ((t16 << 4) & (c.page - 1));
      }
    };
    auto load_k = [&]() {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
#pragma unroll
        for (int j = 0; j < KL; ++j) kx[i][j] = load_once16((const uint8_t*)c.k + row16[i] * RB + koff + 64 * j);
        if constexpr (FP8) {
          ksc[i] = *reinterpret_cast<const f32x4*>(c.k_scale + row16[i] + 4 * g);
          vsc[i] = *reinterpret_cast<const f32x4*>(c.v_scale + row16[i] + 4 * g);
        }
      }
    };
    auto load_v = [&]() {
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int j = 0; j < VL / NS; ++j)
          vx[i * (VL / NS) + j] = load_once16((const uint8_t*)c.v + row16[i] * RB + voff + 1024 * j);
    };
    find_pages(s0);
    load_k();
    load_v();
    for (int s = s0; s < s1; ++s) {
      const int tok0 = s * TOK;
      // S^T: lane = query head r16, registers = tokens 16 i + 4 g + v
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
      auto store_v = [&]() {
#pragma unroll
        for (int j = 0; j < VL; ++j) {
          const int row = j * VR + vrow;
          uint4 u = vx[j];
          if (tail && tok0 + row >= n) u = make_uint4(0, 0, 0, 0);
          if constexpr (FP8) {
            *reinterpret_cast<bf16x8*>(vt + v_slot<HD>(row, 2 * vpc)) = widen8(u.x, u.y);
            *reinterpret_cast<bf16x8*>(vt + v_slot<HD>(row, 2 * vpc + 1)) = widen8(u.z, u.w);
          } else {
            *reinterpret_cast<uint4*>(vt + v_slot<HD>(row, vpc)) = u;
          }
        }
        lds_order();
      };
      f32x4 kss[NS], vss[NS];
      if constexpr (FP8) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          kss[i] = ksc[i] * sc;
          vss[i] = vsc[i];
        }
      }
      // registers go to the next step's loads as soon as they are read
      const bool more = s + 1 < s1;
      if (more) {
        find_pages(s + 1);
        load_k();
      }
      store_v();
      if (more) load_v();
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          x[i][v] *= FP8 ? kss[i][v] : sc;
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
      // O^T += V^T P^T: registers of the two products are the B operand
      bf16x8 pf;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        pf[e] = (__bf16)x[0][e];
        pf[4 + e] = (__bf16)x[1][e];
      }
      const int rlo = 4 * g + (r16 >> 2), rhi = rlo + 16;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int ch = 2 * t + ((r16 & 3) >> 1), b8 = 8 * (r16 & 1);
        const v4i16 lo = lds_read_tr16(reinterpret_cast<const bf16_t*>(vt + v_slot<HD>(rlo, ch) + b8));
        const v4i16 hi = lds_read_tr16(reinterpret_cast<const bf16_t*>(vt + v_slot<HD>(rhi, ch) + b8));
        typedef short v8i16 __attribute__((ext_vector_type(8)));
        const v8i16 vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        acc[t] = mfma16(__builtin_bit_cast(bf16x8, vf), pf, acc[t]);
      }
      lds_order();
    }
    const auto add = [](float a, float b2) { return a + b2; };
    l = xor32_f32(xor16_f32(l, add), add);
    if (bad) l = __builtin_nanf("");  // a page that is none: the sequence's result is NaN
    if (s0 == 0 && s1 == nsteps) {
      if (r16 < nh) {
        const float inv = 1.f / l;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          bf16x4 o;
#pragma unroll
          for (int v = 0; v < 4; ++v) o[v] = (__bf16)(acc[t][v] * inv);
          *reinterpret_cast<bf16x4*>(out + ((long)b * H + hbase + r16) * HD + 16 * t + 4 * g) = o;
        }
      }
    } else {
      const int slot = at == begin ? 0 : 1;
      if (r16 < nh) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
          *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(vt + part_offset<HD>(slot)) + r16 * HD + 16 * t + 4 * g) =
              acc[t];
        if (g == 0) stats[2 * wave + slot][r16] = make_float2(m, l);
      }
      if (lane == 0) seqs[2 * wave + slot] = PartSeq{b, first, nsteps};
    }
    at = first + s1;
    first += nsteps;
    ++b;
    if (at < end) b = list.next(b);  // sequences without tokens hold no step
  }
  __syncthreads();

  // the waves' partials of one sequence, joined: its result where the workgroup
  // held all of it, else the workgroup's partial.  Everything is read up front:
  // one LDS latency, not one for each partial.
  PartSeq ps[8];
  int next[8];  // sequence of the partial behind
#pragma unroll
  for (int e = 0; e < 8; ++e) ps[e] = seqs[e];
  int nb = -1;
#pragma unroll
  for (int e = 7; e >= 0; --e) {
    next[e] = nb;
    if (ps[e].b >= 0) nb = ps[e].b;
  }
  for (int i = tid; i < nh * (HD / 4); i += 256) {
    const int r = i / (HD / 4), f = 4 * (i % (HD / 4));
    float2 st[8];
    f32x4 px[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      st[e] = stats[e][r];
      px[e] = *reinterpret_cast<const f32x4*>(
          reinterpret_cast<const float*>(lds + (e >> 1) * kWaveLds<HD, ROWS> + part_offset<HD>(e & 1)) + r * HD + f);
    }
    float m = kLowest, l = 0.f;
    f32x4 a = f32x4{};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const PartSeq& cur = ps[e];
      if (cur.b < 0) continue;
      const float mn = fmaxf(m, st[e].x), wa = __builtin_amdgcn_exp2f(m - mn),
                  wb = __builtin_amdgcn_exp2f(st[e].x - mn);
      a = a * wa + px[e] * wb;
      l = l * wa + st[e].y * wb;
      m = mn;
      if (next[e] == cur.b) continue;
      if (cur.first >= wg0 && cur.first + cur.steps <= wg1) {
        const float inv = 1.f / l;
        bf16x4 o;
#pragma unroll
        for (int v = 0; v < 4; ++v) o[v] = (__bf16)(a[v] * inv);
        *reinterpret_cast<bf16x4*>(out + ((long)cur.b * H + hbase + r) * HD + f) = o;
      } else {
        const long row = part_row(p, slice, wg, cur.first <= wg0 ? 0 : 1) + r;
        *reinterpret_cast<f32x4*>(part + row * HD + f) = a;
        if (f == 0) stat[row] = make_float2(m, l);
      }
      m = kLowest;
      l = 0.f;
      a = f32x4{};
    }
  }
  // zeros for the sequences without tokens: the workgroup's own, or 64 sequences a wave
  const auto empty = [&](long z) {
    for (int i = lane; i < nh * (HD / 4); i += 64)
      *reinterpret_cast<bf16x4*>(out + (z * H + hbase) * HD + 4 * i) = bf16x4{};
  };
  if (p.whole) {
    if (wg1 == 0 && wave == 0 && wg < c.B) empty(wg);
    return;
  }
  for (int z = (wg * 4 + wave) * 64; z < c.B; z += p.wgs * 256) {
    unsigned long long none = __ballot(z + lane < c.B && list.len(z + lane) == 0);
    for (; none; none &= none - 1) empty(z + __ffsll(none) - 1);
  }
}

// Joins the workgroups' partials of a sequence; nothing where one of them held
// it whole.  Grid (H, B).
template <int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedCacheDims c, const int32_t* __restrict__ lens,
                                                         bf16_t* __restrict__ out, const float* __restrict__ part,
                                                         const float2* __restrict__ stat, const int* __restrict__ starts,
                                                         PagedSplit p) {
  constexpr int TR = HD / 4, NG = 256 / TR;  // threads of a partial; partials read at once
  __shared__ float weight[kPagedMaxWgs];
  __shared__ float red[4];
  __shared__ f32x4 sums[NG][TR];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = blockIdx.x, b = blockIdx.y;
  const int n = StepList{lens, c.B, c.W * c.page}.steps(b);
  if (n == 0) return;
  const int total = starts[c.B], range = max((total + p.wgs - 1) / p.wgs, 1);
  const int first = starts[b], w0 = first / range, w1 = (first + n - 1) / range;
  if (w0 == w1) return;
  const int kvh = h / c.G, hr = h % c.G, slice = kvh * p.head_tiles + hr / kRowsMfma;
  const int count = w1 - w0 + 1;
  // a workgroup's first sequence, unless its range begins before this one
  const auto row = [&](int i) {
    const int w = w0 + i;
    return part_row(p, slice, w, w * range >= first ? 0 : 1) + hr % kRowsMfma;
  };
  const auto block = [&](float x, auto op) {
    x = wave_allreduce_f32(x, op);
    if (lane == 0) red[wave] = x;
    __syncthreads();
    x = op(op(red[0], red[1]), op(red[2], red[3]));
    __syncthreads();
    return x;
  };
  // all that most sequences have is under way at once: a partial a group of
  // threads, a (maximum, sum) or two a thread
  const int gi = tid / TR, f = tid % TR;
  const auto piece = [&](int i) { return *reinterpret_cast<const f32x4*>(part + row(i) * HD + 4 * f); };
  const f32x4 mine = piece(min(gi, count - 1));
  float2 st[kPagedMaxWgs / 256];
  float m = kLowest, l = 0.f;
#pragma unroll
  for (int u = 0; u < kPagedMaxWgs / 256; ++u) {
    const int i = tid + 256 * u;
    st[u] = i < count ? stat[row(i)] : float2{kLowest, 0.f};
    m = fmaxf(m, st[u].x);
  }
  m = block(m, [](float a, float b) { return fmaxf(a, b); });
#pragma unroll
  for (int u = 0; u < kPagedMaxWgs / 256; ++u) {
    const float w = __builtin_amdgcn_exp2f(st[u].x - m);
    weight[tid + 256 * u] = w;
    l += w * st[u].y;
  }
  l = block(l, [](float a, float b) { return a + b; });  // (its barriers are the weights' too)
  f32x4 a = gi < count ? mine * weight[gi] : f32x4{};
#pragma unroll 4
  for (int i = gi + NG; i < count; i += NG) a += piece(i) * weight[i];
  sums[gi][f] = a;
  __syncthreads();
  if (gi) return;
#pragma unroll
  for (int i = 1; i < NG; ++i) a += sums[i][f];
  const float inv = 1.f / l;
  bf16x4 o;
#pragma unroll
  for (int v = 0; v < 4; ++v) o[v] = (__bf16)(a[v] * inv);
  *reinterpret_cast<bf16x4*>(out + ((long)b * c.Hkv * c.G + h) * HD + 4 * f) = o;
}

// A workgroup for each sequence where tables hold at most 16 steps, four for each
// wave, and no second launch (128 sequences of up to 500 tokens, 8 key heads of
// 128: 38 us against 50).  Else the list is cut for two workgroups a CU over all
// slices, and no finer than a step a wave.
// Three or four a CU take longer (three contexts of 65537 .. 131072 tokens, e4m3:
// 124 us with 512 workgroups, 147 with 768, 130 with 1024).
PagedSplit paged_split(const PagedCacheDims& c) {
  PagedSplit p;
  p.head_tiles = (c.G + kRowsMfma - 1) / kRowsMfma;
  p.rows = c.G <= 4 ? 4 : kRowsMfma;
  const long slices = (long)c.Hkv * p.head_tiles;
  const long cap = ((long)c.W * c.page + kPagedStep - 1) / kPagedStep;
  p.whole = cap <= 16;
  p.wgs = (int)(p.whole ? std::max(c.B, 1)
                        : std::max(1L, std::min({512 / slices, (c.B * cap + 3) / 4, (long)kPagedMaxWgs})));
  return p;
}

size_t paged_part_floats(const PagedCacheDims& c, const PagedSplit& p, int hd) {
  return p.whole ? 0 : (size_t)c.Hkv * p.head_tiles * p.wgs * 2 * p.rows * hd;
}

// partials, their (maximum, sum), and each sequence's first step with the number of all behind the last
size_t paged_ws_bytes(const PagedCacheDims& c, int hd) {
  const size_t n = paged_part_floats(c, paged_split(c), hd);
  return n == 0 ? 0 : n * 4 + n / hd * 8 + ((size_t)c.B + 1) * 4;
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
  const PagedSplit p = paged_split(c);
  float* part = (float*)ws;
  const size_t n = paged_part_floats(c, p, hd);
  float2* stat = (float2*)(part + n);
  int* starts = (int*)(stat + n / hd);
  auto run = [&](auto kernel) {
    NAYLIS_TIMED("paged_attn", st,
                 hipLaunchKernelGGL(kernel, dim3(p.wgs, c.Hkv * p.head_tiles), dim3(256), 0, st, c,
                                    (const bf16_t*)q, ldq, hsq, table, lens, (bf16_t*)out, part, stat, starts, p,
                                    scale * kLog2e));
  };
  auto pick = [&](auto rows) {
    constexpr int R = decltype(rows)::value;
    if (hd == 64)
      fp8 ? run(paged_attn_kernel<64, true, R>) : run(paged_attn_kernel<64, false, R>);
    else
      fp8 ? run(paged_attn_kernel<128, true, R>) : run(paged_attn_kernel<128, false, R>);
  };
  p.rows == 4 ? pick(std::integral_constant<int, 4>{}) : pick(std::integral_constant<int, 16>{});
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.whole || p.wgs == 1) return e;
  auto join = [&](auto kernel) {
    NAYLIS_TIMED("paged_join", st,
                 hipLaunchKernelGGL(kernel, dim3(c.Hkv * c.G, c.B), dim3(256), 0, st, c, lens, (bf16_t*)out,
                                    (const float*)part, (const float2*)stat, (const int*)starts, p));
  };
  hd == 64 ? join(paged_join_kernel<64>) : join(paged_join_kernel<128>);
  return hipGetLastError();
}

}  // namespace naylis
