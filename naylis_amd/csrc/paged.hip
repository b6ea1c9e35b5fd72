// Key / value cache in pages, and the attention of a sequence's new tokens over it.
//
// Pages (P, Hkv, page, hd) hold `page` consecutive tokens of one sequence, a
// head's rows together; table (B, W) names each sequence's pages in order.
// Rows are bf16, or e4m3 codes with one fp32 scale per row (the bank's form:
// scale = max|row| / 448, 1 for a row of zeros; code = e4m3(x / scale)), or pairs of
// e2m1 codes with a power of two for 32 features, its exponent in a byte.
//
// Attention: o[b, i, h] = softmax_n(scale q[b, i, h] . k[n]) v[n] over the tokens
// n < lens[b] - (N - 1 - i): the last of N new tokens sees all of its sequence, each one
// before it a token less.  Bound by memory: every live K and V byte is read once
// (again for each further 16 query heads of a key head, or 32 rows of several new
// tokens), past the caches.
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
//
// Several new tokens make more rows of the same products: a row is (token, head), and a
// token's end masks its scores in the steps that reach it.  32 sequences of up to 8191
// tokens, five new ones each, 8 key heads of 128 with four query heads, bf16, 551 MB:
// 99 us (5.6 TB/s; the attention 95, vector units in use 19 % of the time), where one
// call a token would read the cache five times.
//
// Pages of 4 bits: a lane's 16 bytes are 32 features of K, the scale's reach, and widen
// to bf16 by the conversions that take the scale (exact: two bits of a bf16's seven), so
// that products and sums are those of bf16 pages.  64 sequences of up to 4096 tokens,
// one new each, 157 MB: 34.6 us with the join's 4 (5.1 TB/s in the attention); three of
// up to 131072, four new ones each, 385 MB: 76 (5.4 TB/s).  Not the memory alone: a byte
// brings four times the work that it does in bf16, the vector units are in use for half
// the time and LDS for a quarter, and the first loads wait for length and page.
#include "common.h"
#include "launch.h"
#include "packed_tiles.h"
#include "paged_common.h"
#include "timing.h"

#include <algorithm>
#include <type_traits>

namespace naylis {

namespace {

constexpr int kRowsMfma = 16;       // query rows of a product
constexpr int kPagedStep = 32;      // tokens of a step
constexpr int kPagedMaxWgs = 512;   // workgroups that share a slice's steps
constexpr int kJoinFew = 128;       // of them, the most whose partials rows' own threads join

__device__ __forceinline__ f32x4 mfma16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The wave's own LDS writes before its reads, and the other way round: LDS
// serves one wave's accesses in order, so only the compiler has to keep it.
__device__ __forceinline__ void lds_order() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
}

}  // namespace

// New rows into the cache, HD / 8 lanes a row (8191 tokens, 8 heads of 128: bf16 15 us,
// e4m3 18, 4 bits 13.6, of 67, 51 and 43 MB).  Token t goes to sequence
// rows[t] (t itself without rows) at positions[t]; a position or a page outside
// the table or the cache (padding) writes nothing.
template <int HD, PagedFormat FMT>
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
  if constexpr (FMT == kPagedBf16) {
    reinterpret_cast<uint4*>(is_v ? c.v : c.k)[row * LANES + piece] = u;
  } else {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    // the row's lanes are all here: they share t and so every return above
    store_codes<HD, FMT>(c, is_v, row, piece, f);
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

// Whether the partial of a sequence that ends within a wave's range goes to the
// workspace, not to LDS: few waves have one, and of 32 rows, or of 16 beside pages
// of 4 bits, its LDS would leave room for fewer workgroups a CU than the registers do.
constexpr bool ends_outside(PagedFormat f, int rows) { return rows > kRowsMfma || (f == kPagedE2m1 && rows > 4); }

// LDS of a wave: its V tile (32 tokens), where the partial at the end of its range
// goes too (fp32 rows, once the tile is no longer needed), then that of a sequence
// that ends within the range.
template <int HD, PagedFormat FMT, int ROWS>
constexpr int kWaveLds = std::max(32 * 2 * HD, ROWS * HD * 4) + (ends_outside(FMT, ROWS) ? 0 : ROWS * HD * 4);
template <int HD>
__device__ __forceinline__ int part_offset(int slot) {
  static_assert(kRowsMfma * 4 == 32 * 2, "a partial of 16 rows fits the V tile");
  return slot == 0 ? 32 * 2 * HD : 0;
}

// Place of features f .. f + 3 of row r in a wave's partial: a write takes the same
// chunk of sixteen rows, which lie in eight places of the banks.
template <int HD>
__device__ __forceinline__ int part_at(int r, int f) {
  return r * HD + (f ^ (4 * (r & 7)));
}

// Byte of a 16-byte chunk in the V tile: dealt so that the 128 bytes that LDS serves
// at a time lie in its 32 banks once.  A transposing read takes a pair of chunks from
// each of four rows; of widened codes a write takes every second chunk of a row, or of
// e2m1 every fourth one of two (in the halves of a row the chunks of a pair change
// places).
template <int HD, PagedFormat FMT>
__device__ __forceinline__ int v_slot(int row, int chunk) {
  constexpr bool CODES = FMT != kPagedBf16;
  const int f = HD == 128 ? (2 * (row & 7)) ^ (CODES ? chunk >> 3 : 0) : 2 * (row & 3) + (CODES ? row & 1 : 0);
  return row * 2 * HD + ((chunk ^ f) << 4);
}

// Loads past the caches, unless another slice reads the same.
template <bool AGAIN>
__device__ __forceinline__ uint4 load_once16(const uint8_t* p) {
  if constexpr (AGAIN)
    return *reinterpret_cast<const uint4*>(p);
  else
    return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p)));
}
template <int N>
struct Words {
  uint32_t w[N];
};
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <int N, bool AGAIN>
__device__ __forceinline__ Words<N> load_once(const uint8_t* p) {
  using V = std::conditional_t<N == 4, u32x4, u32x2>;
  static_assert(N == 2 || N == 4, "8 or 16 bytes");
  if constexpr (AGAIN)
    return __builtin_bit_cast(Words<N>, *reinterpret_cast<const V*>(p));
  else
    return __builtin_bit_cast(Words<N>, __builtin_nontemporal_load(reinterpret_cast<const V*>(p)));
}

// A query row of a key head is (new token, query head): token-major, so that one
// product's 16 rows see nearly the same keys.
struct Rows {
  int G, N, H;
  __device__ __forceinline__ int token(int row) const { return row / G; }
  // row `row` of key head kvh in out (B, N, H, hd), in heads
  __device__ __forceinline__ long at(int b, int kvh, int row) const {
    return ((long)b * N + row / G) * H + kvh * G + row % G;
  }
};

// Tokens that new token i of a sequence of n sees, where the last of `live` sees
// all; 0 for one that is none or sees nothing.
__device__ __forceinline__ int seen(int n, int live, int i) { return i < live ? max(n - (live - 1 - i), 0) : 0; }

}  // namespace

// partials of (slice, workgroup, 0: the first sequence of its range / 1: the last)
__device__ __forceinline__ long part_row(const PagedSplit& p, int slice, int wg, int slot) {
  return (((long)slice * p.wgs + wg) * 2 + slot) * p.rows;
}

// grid (workgroups of a slice, slices): slice = (key head, 16 or 32 of its query rows).
// A workgroup takes a range of the step list, or (p.whole) the sequence of its
// number, its waves an equal share each.
// ROWS: partials' rows, at least the query rows of a slice; a product's 16 or, of 32,
// two products' for each read of the cache.  MANY: more than one
// new token, or a number of them that each sequence has of its own.  AGAIN: a key head
// has more than one slice, which read the same keys and values at about the same time
// (seven sequences of up to 5775 tokens, 40 rows for each of 4 key heads, bf16: 31 us;
// past the caches 38, and with the choice made in the loop a single slice loses a tenth).
template <int HD, PagedFormat FMT, int ROWS, bool MANY, bool AGAIN = false>
__global__ __launch_bounds__(256, FMT == kPagedE2m1 && ROWS <= kRowsMfma ? 3 : 2) void paged_attn_kernel(
    PagedCacheDims c, PagedQueries q, const int32_t* __restrict__ table, const int32_t* __restrict__ lens,
    bf16_t* __restrict__ out, float* __restrict__ part, float2* __restrict__ stat, int* __restrict__ starts,
    float* __restrict__ ended, PagedSplit p, float sc) {
  constexpr int QT = ROWS > kRowsMfma ? 2 : 1;  // 16-row tiles
  constexpr bool FP8 = FMT == kPagedE4m3, FP4 = FMT == kPagedE2m1;
  constexpr int TOK = kPagedStep;        // tokens of a step
  constexpr int NS = TOK / 16;           // its 16-token products
  constexpr int KS = HD / 32;            // products along the features
  constexpr int NT = HD / 16;            // 16-feature tiles of the output
  constexpr int RB = FP4 ? HD / 2 : FP8 ? HD : 2 * HD;  // bytes of a cache row
  constexpr int KL = FP4 ? 1 : RB / 64;  // 16-byte loads of a lane for 16 tokens of K
  constexpr int VR = FP4 ? 16 : 1024 / RB;  // rows of V that a load of 64 lanes covers
  constexpr int VL = TOK / VR;           // such loads
  constexpr int NW = HD / 32;            // 4 bits: words of such a load, HD / 4 features
  __shared__ __align__(16) uint8_t lds[4 * kWaveLds<HD, FMT, ROWS>];
  __shared__ PartSeq seqs[8];
  __shared__ float2 stats[8][ROWS];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint8_t* vt = lds + wave * kWaveLds<HD, FMT, ROWS>;
  const int wg = blockIdx.x, slice = blockIdx.y;
  const int kvh = slice / p.head_tiles, h0 = QT * kRowsMfma * (slice % p.head_tiles);
  const int nh = min(QT * kRowsMfma, (MANY ? c.G * c.N : c.G) - h0);  // live query rows of the slice
  constexpr bool OUTSIDE = ends_outside(FMT, ROWS);
  // the partial that ends within a wave's range
  if constexpr (OUTSIDE) ended += ((long)slice * p.wgs + wg) * 4 * ROWS * HD;
  const int H = c.Hkv * c.G, hbase = kvh * c.G + h0;
  const Rows rows{c.G, c.N, H};
  // the slice's row r of sequence b in out
  const auto out_row = [&](long b, int r) {
    return out + (MANY ? rows.at((int)b, kvh, h0 + r) : b * H + hbase + r) * HD;
  };
  const auto live_of = [&](int b) { return q.live ? min(max(q.live[b], 0), c.N) : c.N; };
  // whether the slice's row r sees no token of sequence b
  const auto blind = [&](int b, int r) { return MANY && seen(lens[b], live_of(b), rows.token(h0 + r)) == 0; };
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
  // bytes of a lane's loads.  V: row vrow, piece vpc; K: row r16, pieces g, g + 4, ..
  const uint32_t voff = lane * (FP4 ? 4 * NW : 16), koff = r16 * RB + g * (FP4 ? 4 * NW : 16);
  const uint32_t veoff = lane * NW / 4, keoff = r16 * NW + g * NW / 4;
  const int vrow = FP4 ? lane / 4 : lane / (RB / 16), vpc = FP4 ? lane % 4 : lane % (RB / 16);

  while (at < end && b < c.B) {
    const int n = list.len(b), nsteps = (n + TOK - 1) / TOK;
    const int s0 = at - first, s1 = min(end - first, nsteps);  // this wave's steps of sequence b
    bool bad = lens[b] > list.cap;                             // longer than its table
    // tokens that the lane's row sees, and the fewest that one does
    const int live = MANY ? live_of(b) : 1, all = n - (live - 1);
    int mine[QT];
#pragma unroll
    for (int u = 0; u < QT; ++u) mine[u] = MANY ? n - max(live - 1 - rows.token(h0 + 16 * u + r16), 0) : n;
    if (!p.whole && s0 == 0 && slice == 0 && lane == 0) starts[b] = first;

    bf16x8 qf[QT][KS];
#pragma unroll
    for (int u = 0; u < QT; ++u) {
      const int row = h0 + min(16 * u + r16, nh - 1);
      const bf16_t* qp = (const bf16_t*)q.q + (long)b * q.ldb +
                         (MANY ? rows.token(row) * q.ldt + (long)(kvh * c.G + row % c.G) * q.hs
                               : (long)(kvh * c.G + row) * q.hs);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        // feature order of the products: as the lane's 16-byte pieces of K hold them
        const int f = FP4   ? 8 * NW * g + 8 * ks
                      : FP8 ? 64 * (ks >> 1) + 16 * g + 8 * (ks & 1)
                            : 32 * ks + 8 * g;
        qf[u][ks] = *reinterpret_cast<const bf16x8*>(qp + f);
        if (16 * u + r16 >= nh) qf[u][ks] = bf16x8{};
      }
    }
    f32x4 acc[QT][NT];
    float m[QT], l[QT];
#pragma unroll
    for (int u = 0; u < QT; ++u) {
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[u][t] = f32x4{};
      m[u] = kLowest;
      l[u] = 0.f;
    }

    uint4 kx[NS][KL], vx[VL];
    Words<NW> kw[NS], vw[NS];  // 4 bits
    uint32_t ke[NS], ve[NS];   // their scales' exponents
    f32x4 ksc[NS], vsc[NS];    // scales of tokens 16 i + 4 g ..
    long row16[NS];          // cache row of each 16-token group of the step being loaded
    // pages a step ahead, by scalar loads: a wait for them leaves the rows' loads in
    // flight.  Groups past the end take the last token's page, and nothing of it counts.
    const int32_t* pages = table + (long)b * c.W;
    int ids[NS];
    auto fetch_pages = [&](int step) {
#pragma unroll
      for (int i = 0; i < NS; ++i) ids[i] = pages[min((step * NS + i) << 4, n - 1) >> shift];
    };
    auto take_pages = [&](int step) {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        int id = ids[i];
        if (!page_ok(id, c.P)) {
          bad = true;
          id = 0;
        }
        row16[i] = ((long)id * c.Hkv + kvh) * c.page + (((step * NS + i) << 4) & (c.page - 1));
      }
    };
    // (a lane's offset is new to the compiler each time, so that the uniform part of
    // an address stays in scalar registers)
    const auto lane_offset = [](uint32_t x) {
      asm("" : "+v"(x));
      return x;
    };
    auto load_k = [&]() {
      const uint32_t off = lane_offset(koff), eoff = lane_offset(keoff);
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        if constexpr (FP4) {
          kw[i] = load_once<NW, AGAIN>((const uint8_t*)c.k + row16[i] * RB + off);
          ke[i] = __builtin_nontemporal_load((const uint8_t*)c.k_scale + row16[i] * NW + eoff);
        } else {
#pragma unroll
          for (int j = 0; j < KL; ++j)
            kx[i][j] = load_once16<AGAIN>((const uint8_t*)c.k + row16[i] * RB + 64 * j + off);
        }
        if constexpr (FP8) {
          ksc[i] = *reinterpret_cast<const f32x4*>((const float*)c.k_scale + row16[i] + 4 * g);
          vsc[i] = *reinterpret_cast<const f32x4*>((const float*)c.v_scale + row16[i] + 4 * g);
        }
      }
    };
    auto load_v = [&]() {
      const uint32_t off = lane_offset(voff), eoff = lane_offset(veoff);
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        if constexpr (FP4) {
          vw[i] = load_once<NW, AGAIN>((const uint8_t*)c.v + row16[i] * RB + off);
          ve[i] = __builtin_nontemporal_load((const uint8_t*)c.v_scale + row16[i] * NW + eoff);
        } else {
#pragma unroll
          for (int j = 0; j < VL / NS; ++j)
            vx[i * (VL / NS) + j] = load_once16<AGAIN>((const uint8_t*)c.v + row16[i] * RB + 1024 * j + off);
        }
      }
    };
    fetch_pages(s0);
    take_pages(s0);
    fetch_pages(s0 + 1);
    load_k();
    load_v();
    for (int s = s0; s < s1; ++s) {
      const int tok0 = s * TOK;
      // S^T: lane = query head r16, registers = tokens 16 i + 4 g + v
      f32x4 x[QT][NS];
#pragma unroll
      for (int i = 0; i < NS; ++i) {
#pragma unroll
        for (int u = 0; u < QT; ++u) x[u][i] = f32x4{};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          bf16x8 kf;
          if constexpr (FP4) {
            kf = widen8_e2m1(kw[i].w[ks], ke[i]);
          } else if constexpr (FP8) {
            const uint4 u = kx[i][ks >> 1];
            kf = (ks & 1) ? widen8(u.z, u.w) : widen8(u.x, u.y);
          } else {
            kf = __builtin_bit_cast(bf16x8, kx[i][ks]);
          }
#pragma unroll
          for (int u = 0; u < QT; ++u) x[u][i] = mfma16(kf, qf[u][ks], x[u][i]);
        }
      }
      const bool tail = tok0 + TOK > (MANY ? all : n);
      // V rows to LDS as bf16; rows past the sequence as zeros, whatever the page holds there
      auto store_v = [&]() {
        if constexpr (FP4) {
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            const int row = 16 * i + vrow;
            if (tail && tok0 + row >= n) {
              vw[i] = Words<NW>{};
              ve[i] = 127;
            }
#pragma unroll
            for (int w = 0; w < NW; ++w)
              *reinterpret_cast<bf16x8*>(vt + v_slot<HD, FMT>(row, NW * vpc + w)) = widen8_e2m1(vw[i].w[w], ve[i]);
          }
          lds_order();
          return;
        }
#pragma unroll
        for (int j = 0; j < VL; ++j) {
          const int row = j * VR + vrow;
          if (tail && tok0 + row >= n) vx[j] = make_uint4(0, 0, 0, 0);
          const uint4 u = vx[j];
          if constexpr (FP8) {
            *reinterpret_cast<bf16x8*>(vt + v_slot<HD, FMT>(row, 2 * vpc)) = widen8(u.x, u.y);
            *reinterpret_cast<bf16x8*>(vt + v_slot<HD, FMT>(row, 2 * vpc + 1)) = widen8(u.z, u.w);
          } else {
            *reinterpret_cast<uint4*>(vt + v_slot<HD, FMT>(row, vpc)) = u;
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
        take_pages(s + 1);
        fetch_pages(s + 2);
        load_k();
      }
      store_v();
      if (more) load_v();
#pragma unroll
      for (int u = 0; u < QT; ++u) {
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int v = 0; v < 4; ++v) x[u][i][v] = mul_rn(x[u][i][v], FP8 ? kss[i][v] : sc);
        if (__builtin_expect(tail, 0))
#pragma unroll
          for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v)
              if (tok0 + 16 * i + 4 * g + v >= mine[u]) x[u][i][v] = -INFINITY;
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int v = 0; v < 4; ++v) mx = fmaxf(mx, x[u][i][v]);
        const auto fmx = [](float a, float b) { return fmaxf(a, b); };
        mx = xor32_f32(xor16_f32(mx, fmx), fmx);
        const float mn = fmaxf(m[u], mx), al = __builtin_amdgcn_exp2f(m[u] - mn);
        // (times 1 where no row has a new maximum)
        if (__any(mn > m[u])) {
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[u][t] *= al;
        }
        m[u] = mn;
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            x[u][i][v] = __builtin_amdgcn_exp2f(x[u][i][v] - mn);
            l[u] = i + v ? l[u] + x[u][i][v] : __builtin_fmaf(l[u], al, x[u][i][v]);
            if constexpr (FP8) x[u][i][v] *= vss[i][v];
          }
        // rows past the end: their weight is 0, their scale may be anything
        if (FP8 && __builtin_expect(tail, 0))
#pragma unroll
          for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v)
              if (tok0 + 16 * i + 4 * g + v >= mine[u]) x[u][i][v] = 0.f;
      }
      // O^T += V^T P^T: registers of the two products are the B operand
      bf16x8 pf[QT];
#pragma unroll
      for (int u = 0; u < QT; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pf[u][e] = (__bf16)x[u][0][e];
          pf[u][4 + e] = (__bf16)x[u][1][e];
        }
      const int rlo = 4 * g + (r16 >> 2), rhi = rlo + 16;
      typedef short v8i16 __attribute__((ext_vector_type(8)));
      v8i16 vf[NT];
      const auto read_v = [&](int t) {
        const int ch = 2 * t + ((r16 & 3) >> 1), b8 = 8 * (r16 & 1);
        const v4i16 lo = lds_read_tr16(reinterpret_cast<const bf16_t*>(vt + v_slot<HD, FMT>(rlo, ch) + b8));
        const v4i16 hi = lds_read_tr16(reinterpret_cast<const bf16_t*>(vt + v_slot<HD, FMT>(rhi, ch) + b8));
        vf[t] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      };
      // (of two tiles of rows the reads are kept AHEAD products in front, where the
      // compiler, short of registers, waits for each: with the partials' places 56 -> 53.5
      // us for 32 sequences of up to 8191 tokens in 4 bits, eight new ones each)
      constexpr int AHEAD = QT > 1 ? 2 : 0;
#pragma unroll
      for (int t = 0; t < AHEAD; ++t) read_v(t);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t + AHEAD < NT) read_v(t + AHEAD);
        if constexpr (AHEAD > 0) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < QT; ++u) acc[u][t] = mfma16(__builtin_bit_cast(bf16x8, vf[t]), pf[u], acc[u][t]);
        if constexpr (AHEAD > 0) __builtin_amdgcn_sched_barrier(0);
      }
      lds_order();
    }
    const auto add = [](float a, float b2) { return a + b2; };
    const bool whole = s0 == 0 && s1 == nsteps;
    const int slot = first + s1 < end ? 0 : 1;  // ends within the range, or with it
    // (new to the compiler here, so that the places keep no registers through the steps)
    int lane_p = lane;
    asm volatile("" : "+v"(lane_p));
#pragma unroll
    for (int u = 0; u < QT; ++u) {
      const int r = 16 * u + r16, rp = 16 * u + (lane_p & 15), gp = lane_p >> 4;
      l[u] = xor32_f32(xor16_f32(l[u], add), add);
      if (bad) l[u] = __builtin_nanf("");  // a page that is none: the sequence's result is NaN
      if (r >= nh) continue;
      if (whole) {
        const float inv = 1.f / l[u];
        const bool none = blind(b, r);
        bf16_t* to = out_row(b, r);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          bf16x4 o;
#pragma unroll
          for (int v = 0; v < 4; ++v) o[v] = (__bf16)(none ? 0.f : acc[u][t][v] * inv);
          *reinterpret_cast<bf16x4*>(to + 16 * t + 4 * g) = o;
        }
      } else {
        float* to = OUTSIDE && slot == 0 ? ended + (long)wave * ROWS * HD
                                         : reinterpret_cast<float*>(vt + part_offset<HD>(slot));
#pragma unroll
        for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4*>(to + part_at<HD>(rp, 16 * t + 4 * gp)) = acc[u][t];
        if (g == 0) stats[2 * wave + slot][r] = make_float2(m[u], l[u]);
      }
    }
    if (!whole && lane == 0) seqs[2 * wave + slot] = PartSeq{b, first, nsteps};
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
      if (OUTSIDE && e % 2 == 0) {
        if (ps[e].b >= 0) px[e] = *reinterpret_cast<const f32x4*>(ended + (e >> 1) * ROWS * HD + part_at<HD>(r, f));
      } else {
        px[e] = *reinterpret_cast<const f32x4*>(
            reinterpret_cast<const float*>(lds + (e >> 1) * kWaveLds<HD, FMT, ROWS> + part_offset<HD>(e & 1)) +
            part_at<HD>(r, f));
      }
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
        const bool none = blind(cur.b, r);
        bf16x4 o;
#pragma unroll
        for (int v = 0; v < 4; ++v) o[v] = (__bf16)(none ? 0.f : a[v] * inv);
        *reinterpret_cast<bf16x4*>(out_row(cur.b, r) + f) = o;
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
      *reinterpret_cast<bf16x4*>(out_row(z, i / (HD / 4)) + 4 * (i % (HD / 4))) = bf16x4{};
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
// it whole.  Grid (N H, B).
template <int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedCacheDims c, const int32_t* __restrict__ live,
                                                         const int32_t* __restrict__ lens, bf16_t* __restrict__ out,
                                                         const float* __restrict__ part, const float2* __restrict__ stat,
                                                         const int* __restrict__ starts, PagedSplit p) {
  constexpr int TR = HD / 4, NG = 256 / TR;  // threads of a partial; partials read at once
  __shared__ float weight[kPagedMaxWgs];
  __shared__ float red[4];
  __shared__ f32x4 sums[NG][TR];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int H = c.Hkv * c.G, token = blockIdx.x / H, h = blockIdx.x % H, b = blockIdx.y;
  const StepList list{lens, c.B, c.W * c.page};
  const int n = list.steps(b);
  if (n == 0) return;
  const int total = starts[c.B], range = max((total + p.wgs - 1) / p.wgs, 1);
  const int first = starts[b], w0 = first / range, w1 = (first + n - 1) / range;
  if (w0 == w1) return;
  const int kvh = h / c.G, hr = token * c.G + h % c.G, slice = kvh * p.head_tiles + hr / p.tile;
  const int count = w1 - w0 + 1;
  // a workgroup's first sequence, unless its range begins before this one
  const auto row = [&](int i) {
    const int w = w0 + i;
    return part_row(p, slice, w, w * range >= first ? 0 : 1) + hr % p.tile;
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
  const bool none = seen(lens[b], live ? min(max(live[b], 0), c.N) : c.N, token) == 0;
  const float inv = 1.f / l;
  bf16x4 o;
#pragma unroll
  for (int v = 0; v < 4; ++v) o[v] = (__bf16)(none ? 0.f : a[v] * inv);
  *reinterpret_cast<bf16x4*>(out + (((long)b * c.N + token) * H + h) * HD + 4 * f) = o;
}

// The same with HD / 4 threads a row, for few partials of many rows: one after another,
// or for a long sequence among short ones (its length stays on the device) the weights
// first, a partial a thread, and then kRun rows at a time.  Grid (1024 / HD rows of a key
// head, key heads, B).
template <int HD>
__global__ __launch_bounds__(256) void paged_join_few_kernel(PagedCacheDims c, const int32_t* __restrict__ live,
                                                             const int32_t* __restrict__ lens, bf16_t* __restrict__ out,
                                                             const float* __restrict__ part,
                                                             const float2* __restrict__ stat,
                                                             const int* __restrict__ starts, PagedSplit p) {
  constexpr int TR = HD / 4, NG = 256 / TR, kRun = 16;
  static_assert(kJoinFew % TR == 0 && kJoinFew % kRun == 0, "whole rounds");
  __shared__ float weights[NG][kJoinFew];
  const int hr = blockIdx.x * NG + threadIdx.x / TR, f = threadIdx.x % TR, kvh = blockIdx.y, b = blockIdx.z;
  const StepList list{lens, c.B, c.W * c.page};
  const int n = list.steps(b);
  if (n == 0 || hr >= c.G * c.N) return;
  const int total = starts[c.B], range = max((total + p.wgs - 1) / p.wgs, 1);
  const int first = starts[b], w0 = first / range, w1 = (first + n - 1) / range;
  if (w0 == w1) return;
  const int slice = kvh * p.head_tiles + hr / p.tile, count = w1 - w0 + 1;
  const auto row = [&](int w) { return part_row(p, slice, w, w * range >= first ? 0 : 1) + hr % p.tile; };
  const auto piece = [&](int w) { return *reinterpret_cast<const f32x4*>(part + row(w) * HD + 4 * f); };
  float m = kLowest, l = 0.f;
  f32x4 a = f32x4{};
  if (count <= kRun) {
#pragma unroll 4
    for (int w = w0; w <= w1; ++w) {
      const float2 s = stat[row(w)];
      const f32x4 x = piece(w);
      const float mn = fmaxf(m, s.x), wa = __builtin_amdgcn_exp2f(m - mn), wb = __builtin_amdgcn_exp2f(s.x - mn);
      a = a * wa + x * wb;
      l = l * wa + s.y * wb;
      m = mn;
    }
  } else {
    // (of a row's own threads, which lie in one wave)
    float* weight = weights[threadIdx.x / TR];
    float2 st[kJoinFew / TR];
#pragma unroll
    for (int u = 0; u < kJoinFew / TR; ++u) {
      const int i = f + TR * u;
      st[u] = i < count ? stat[row(w0 + i)] : float2{kLowest, 0.f};
      m = fmaxf(m, st[u].x);
    }
#pragma unroll
    for (int o = 1; o < TR; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
#pragma unroll
    for (int u = 0; u < kJoinFew / TR; ++u) {
      const int i = f + TR * u;
      const float w = i < count ? __builtin_amdgcn_exp2f(st[u].x - m) : 0.f;
      weight[i] = w;
      l += w * st[u].y;
    }
#pragma unroll
    for (int o = 1; o < TR; o <<= 1) l += __shfl_xor(l, o, 64);
    lds_order();
    for (int i0 = 0; i0 < count; i0 += kRun) {
      f32x4 x[kRun];
#pragma unroll
      for (int i = 0; i < kRun; ++i) x[i] = piece(w0 + min(i0 + i, count - 1));
#pragma unroll
      for (int i = 0; i < kRun; ++i) a += x[i] * weight[i0 + i];
    }
  }
  const int token = hr / c.G;
  const bool none = seen(lens[b], live ? min(max(live[b], 0), c.N) : c.N, token) == 0;
  const float inv = 1.f / l;
  bf16x4 o;
#pragma unroll
  for (int v = 0; v < 4; ++v) o[v] = (__bf16)(none ? 0.f : a[v] * inv);
  *reinterpret_cast<bf16x4*>(out + Rows{c.G, c.N, c.Hkv * c.G}.at(b, kvh, hr) * HD + 4 * f) = o;
}

// A workgroup for each sequence where tables hold at most 16 steps, four for each
// wave, and no second launch (128 sequences of up to 500 tokens, 8 key heads of
// 128: 38 us against 50), and in the forms with several tokens or 4 bits, whose
// partials are more of the work, at most 32 steps where these workgroups are one round
// of the chip or a good part of one (32 sequences of up to 1000 tokens, four new ones, 8
// key heads of 128 with four query heads, us whole and cut: bf16 21 and 25, e4m3 18 and
// 22, 4 bits 14 and 20; of 8 sequences 17.4 and 17.0, 15.9 and 16.5, 14 and 16, of one 15
// and 12, 18 and 12, 14 and 12; of 128 69 and 58, 46 and 40, 34 and 34).  Else the list is
// cut for two workgroups a CU over all slices, and no finer than a step a wave.
// Three or four a CU take longer (three contexts of 65537 .. 131072 tokens, e4m3:
// 124 us with 512 workgroups, 147 with 768, 130 with 1024); pages of 4 bits, with
// half the loads of a step, leave registers for three and gain by them (three
// contexts of 99396 .. 131072 tokens, four new ones each: 71 us against 76).  Several
// tokens over bf16 pages take one workgroup a CU, whose waves have 64 KB under way, for
// half the partials (32 sequences of up to 8191 tokens, five new ones each: 99 us against
// 105; two 101 against 104; e4m3 in turn 77 against 70).  Heads of 64 have half of that
// under way but gain alike where a key head has more rows than four (five tokens of four
// query heads, the same sequences 62.4 and 62.5, 64 of up to 2048 tokens and two key heads
// 19.0 and 21.5, one of 30000 20.6 and 22.1); of up to four rows they lose a little (the
// same 58.0 and 57.2, 15.3 and 14.8, 18.1 and 18.4), where heads of 128 do not (103 and
// 106, 21.3 and 20.8, 31 and 33).
PagedSplit paged_split(const PagedCacheDims& c, PagedFormat fmt) {
  PagedSplit p;
  const int rows = c.G * c.N;
  // several tokens' rows beyond a product's go two products a read of the cache
  p.tile = c.N > 1 && rows > kRowsMfma ? 2 * kRowsMfma : kRowsMfma;
  p.head_tiles = (rows + p.tile - 1) / p.tile;
  p.rows = rows <= 4 ? 4 : p.tile;
  const long slices = (long)c.Hkv * p.head_tiles;
  const long cap = ((long)c.W * c.page + kPagedStep - 1) / kPagedStep;
  const long most = fmt == kPagedE2m1 && p.tile == kRowsMfma ? 768 : 512;
  p.whole = cap <= 16 || ((c.N > 1 || fmt == kPagedE2m1) && cap <= 32 && c.B * slices >= 64 && c.B * slices <= most);
  const long cut = fmt == kPagedBf16 && c.N > 1 ? 256 : most;
  p.wgs = (int)(p.whole ? std::max(c.B, 1)
                        : std::max(1L, std::min({cut / slices, (c.B * cap + 3) / 4, (long)kPagedMaxWgs})));
  return p;
}

// Several tokens, or pages of 4 bits, of sequences that have eight partials each or so
// on average: a launch of a thousand workgroups less takes a microsecond less, of several
// thousand more (64 sequences of up to 4096 tokens, four query heads of 128 a key head, us
// with it and with the other join: eight key heads, five tokens, bf16 112 and 121, e4m3 82
// and 91; one token, 4 bits 37 and 39).  One of them may have all there are, which the
// other join reads by more threads (100000 tokens among 63 sequences of up to 120: 101 and
// 103, 93 and 93, 40 and 35; two key heads, bf16, 128 partials, 45 and 39, where even
// sequences take 38 and 40; four, 4 bits, 192 partials, 35 and 25, even ones 25 and 25).
// (One token over other pages keeps the order of its sums.)
bool paged_join_few(const PagedCacheDims& c, const PagedSplit& p, PagedFormat fmt) {
  return (c.N > 1 || fmt == kPagedE2m1) && p.wgs <= std::min(8 * c.B, kJoinFew);
}

size_t paged_part_floats(const PagedCacheDims& c, const PagedSplit& p, int hd) {
  return p.whole ? 0 : (size_t)c.Hkv * p.head_tiles * p.wgs * 2 * p.rows * hd;
}

// partials, their (maximum, sum), and each sequence's first step with the number of all behind the last
size_t paged_joined_bytes(const PagedCacheDims& c, const PagedSplit& p, int hd) {
  const size_t n = paged_part_floats(c, p, hd);
  return n == 0 ? 0 : n * 4 + n / hd * 8 + (((size_t)c.B + 1) * 4 + 15) / 16 * 16;
}

// and where they are outside LDS, the partials that end within a wave's range
size_t paged_ws_bytes(const PagedCacheDims& c, int hd, PagedFormat fmt) {
  const PagedSplit p = paged_split(c, fmt);
  return paged_joined_bytes(c, p, hd) + (ends_outside(fmt, p.rows) ? paged_part_floats(c, p, hd) * 2 * 4 : 0);
}

hipError_t launch_paged_append(const PagedCacheDims& c, int hd, PagedFormat fmt, const void* k, const void* v,
                               const int32_t* table, const int32_t* positions, const int32_t* rows,
                               const PagedNew& src, hipStream_t st) {
  const long threads = src.T * c.Hkv * 2 * (hd / 8);
  with_format(hd, fmt, [&](auto d, auto f) {
    NAYLIS_TIMED("paged_append", st,
                 hipLaunchKernelGGL((paged_append_kernel<decltype(d)::value, decltype(f)::value>),
                                    dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, c, (const bf16_t*)k,
                                    (const bf16_t*)v, table, positions, rows, src));
  });
  return hipGetLastError();
}

hipError_t launch_paged_attn(const PagedCacheDims& c, int hd, PagedFormat fmt, const PagedQueries& q,
                             const int32_t* table, const int32_t* lens, void* out, void* ws, float scale,
                             hipStream_t st) {
  const PagedSplit p = paged_split(c, fmt);
  float* part = (float*)ws;
  const size_t n = paged_part_floats(c, p, hd);
  float2* stat = (float2*)(part + n);
  int* starts = (int*)(stat + n / hd);
  float* ended = (float*)((char*)ws + paged_joined_bytes(c, p, hd));
  auto run = [&](auto kernel) {
    NAYLIS_TIMED("paged_attn", st,
                 hipLaunchKernelGGL(kernel, dim3(p.wgs, c.Hkv * p.head_tiles), dim3(256), 0, st, c, q, table, lens,
                                    (bf16_t*)out, part, stat, starts, ended, p, scale * kLog2e));
  };
  with_format(hd, fmt, [&](auto d, auto f) {
    constexpr int HD = decltype(d)::value;
    constexpr PagedFormat F = decltype(f)::value;
    if (c.N > 1 || q.live)
      p.rows == 4    ? run(paged_attn_kernel<HD, F, 4, true>)
      : p.rows == 16 ? run(paged_attn_kernel<HD, F, 16, true>)
      : p.head_tiles == 1 ? run(paged_attn_kernel<HD, F, 32, true>)
                          : run(paged_attn_kernel<HD, F, 32, true, true>);
    else
      p.rows == 4 ? run(paged_attn_kernel<HD, F, 4, false>) : run(paged_attn_kernel<HD, F, 16, false>);
  });
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.whole || p.wgs == 1) return e;
  auto join = [&](auto kernel, dim3 grid) {
    NAYLIS_TIMED("paged_join", st,
                 hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, c, q.live, lens, (bf16_t*)out, (const float*)part,
                                    (const float2*)stat, (const int*)starts, p));
  };
  if (paged_join_few(c, p, fmt)) {
    const dim3 grid((c.G * c.N * hd + 1023) / 1024, c.Hkv, c.B);
    hd == 64 ? join(paged_join_few_kernel<64>, grid) : join(paged_join_few_kernel<128>, grid);
  } else {
    const dim3 grid(c.Hkv * c.G * c.N, c.B);
    hd == 64 ? join(paged_join_kernel<64>, grid) : join(paged_join_kernel<128>, grid);
  }
  return hipGetLastError();
}

}  // namespace naylis
