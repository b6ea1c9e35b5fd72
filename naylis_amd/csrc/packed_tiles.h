// Which tile of which packed sequence a workgroup takes (packed attention).
//
// Sequences are given by their offsets alone, which are on the device, so the
// grid has the most tiles that T rows in n sequences can have, and a workgroup's
// first wave finds its tile from the offsets: no plan to build, nothing to
// copy, no extra launch.  Tiles are ranked by their work, in levels of 128
// rows of the other operand, longest first: F(x) = number of tiles with more
// than x rows is a sum over the sequences (one wave reduction), so a binary
// search over x finds a rank's level and one scan over the sequences its
// tile.  About 0.5 us of a workgroup's time for up to 62 sequences (their
// offsets stay in registers); more of them are read again at every step.
//
// The rows before the first offset and behind the last one are sequences 0
// and n + 1, without anything to attend to: their results are zeros.  Offsets
// are clamped to [0, T], so that no contents of the arrays reach outside the
// tensors; what falls in descending offsets is unspecified.
#pragma once
#include "common.h"
#include "launch.h"

namespace naylis {

constexpr int kTileRows = 128;

// most tiles of `tile` rows that `rows` rows in n sequences have, the two outer ranges included
inline long packed_tiles(long rows, long n, int tile = kTileRows) { return (rows + (tile - 1) * (n + 2)) / tile; }

struct PackedTile {
  int q0, lq, k0, lk;  // the sequence: first rows and lengths
  int block;           // tile index within its sequence
  bool live;
};

__device__ __forceinline__ int wave_allsum_i32(int x) {
  x += dpp_i32<0xb1>(x);
  x += dpp_i32<0x4e>(x);
  x += dpp_i32<0x141>(x);
  x += dpp_i32<0x140>(x);
  auto r = __builtin_amdgcn_permlane16_swap((unsigned)x, (unsigned)x, false, false);
  x = (int)r[0] + (int)r[1];
  r = __builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)x, false, false);
  return (int)r[0] + (int)r[1];
}

struct PackedSpan {
  int q0, lq, k0, lk;
};

__device__ __forceinline__ PackedSpan packed_span(const PackedSeqs& s, int i) {
  PackedSpan p{0, 0, 0, 0};
  if (i > s.n + 1) return p;
  const int lo = max(i - 1, 0), hi = min(i, s.n);
  const int qa = i == 0 ? 0 : min(max(s.cu_q[lo], 0), s.T), qb = i > s.n ? s.T : min(max(s.cu_q[hi], 0), s.T);
  const int ka = i == 0 ? 0 : min(max(s.cu_k[lo], 0), s.Tk), kb = i > s.n ? s.Tk : min(max(s.cu_k[hi], 0), s.Tk);
  p.q0 = qa;
  p.lq = max(qb - qa, 0);
  p.k0 = ka;
  p.lk = max(kb - ka, 0);
  return p;
}

// Tiles of one sequence with work over x (x < 0: all of them).  Query tiles
// (KEYS false): work = keys that the tile's last query sees, growing with the
// tile.  Key tiles: work = queries that see the tile's first key, falling with
// the tile.  The outer ranges have no work.
template <bool KEYS, int TILE>
__device__ __forceinline__ int tiles_over(const PackedSpan& p, bool outer, int x) {
  const int rows = KEYS ? p.lk : p.lq, all = (rows + TILE - 1) / TILE;
  if (x < 0) return all;
  if (outer) return 0;
  if (KEYS) return p.lq <= x ? 0 : min(all, max(0, (p.lk - x + TILE - 1) / TILE));
  const int y = x - p.lk + p.lq;  // tiles whose end min(lq, (j + 1) rows) lies over y
  return y < 0 ? all : y >= p.lq ? 0 : all - y / TILE;
}

template <bool KEYS, int TILE>
__device__ __forceinline__ PackedTile search_tile(const PackedSeqs& s, int rank) {
  const int lane = threadIdx.x & 63, count = s.n + 2;
  const PackedSpan mine = packed_span(s, lane);
  const auto outer = [&](int i) { return i == 0 || i == s.n + 1; };
  const auto total = [&](int x) {
    int t = tiles_over<KEYS, TILE>(mine, outer(lane), x);
    for (int base = 64; base < count; base += 64)
      t += tiles_over<KEYS, TILE>(packed_span(s, base + lane), outer(base + lane), x);
    return __builtin_amdgcn_readfirstlane(wave_allsum_i32(t));
  };
  PackedTile tile{0, 0, 0, 0, 0, false};
  if (rank >= total(-1)) return tile;
  // the first level whose work no tile before `rank` lies under: F(128 lo) <= rank
  int most = KEYS ? mine.lq : mine.lk;
  for (int base = 64; base < count; base += 64) {
    const PackedSpan p = packed_span(s, base + lane);
    most = max(most, KEYS ? p.lq : p.lk);
  }
  int lo = 0, hi = (-wave_allmin_i32(-most) + kTileRows - 1) / kTileRows;
  hi = __builtin_amdgcn_readfirstlane(hi);
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (total(mid * kTileRows) <= rank)
      hi = mid;
    else
      lo = mid + 1;
  }
  const int x = lo * kTileRows, above = lo == 0 ? -1 : x - kTileRows;
  int left = rank - total(x);
  for (int base = 0; base < count; base += 64) {
    const PackedSpan p = base == 0 ? mine : packed_span(s, base + lane);
    const int over = tiles_over<KEYS, TILE>(p, outer(base + lane), x);
    const int here = tiles_over<KEYS, TILE>(p, outer(base + lane), above) - over;
    int sum = here;  // inclusive scan
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int t = __shfl_up(sum, o, 64);
      if (lane >= o) sum += t;
    }
    const unsigned long long past = __ballot(sum > left);
    if (past) {
      const int src = __ffsll(past) - 1;
      const int nth = left - __builtin_amdgcn_readlane(sum - here, src), o = __builtin_amdgcn_readlane(over, src);
      tile.q0 = __builtin_amdgcn_readlane(p.q0, src);
      tile.lq = __builtin_amdgcn_readlane(p.lq, src);
      tile.k0 = __builtin_amdgcn_readlane(p.k0, src);
      tile.lk = __builtin_amdgcn_readlane(p.lk, src);
      if (base + src == 0 || base + src == s.n + 1) (KEYS ? tile.lq : tile.lk) = 0;
      const int all = ((KEYS ? tile.lk : tile.lq) + TILE - 1) / TILE;
      tile.block = KEYS ? o + nth : all - 1 - o - nth;
      tile.live = tile.block >= 0 && tile.block < all;
      return tile;
    }
    left -= __builtin_amdgcn_readlane(sum, 63);
  }
  return tile;
}

// The workgroup's tile: searched by its first wave alone (the others' vector
// units would do the same 300 instructions for nothing).
template <bool KEYS, int TILE = kTileRows>
__device__ __forceinline__ PackedTile find_tile(const PackedSeqs& s, int rank) {
  __shared__ PackedTile found;
  if (threadIdx.x < 64) {
    const PackedTile t = search_tile<KEYS, TILE>(s, rank);
    if (threadIdx.x == 0) found = t;
  }
  __syncthreads();
  PackedTile t = found;
  t.q0 = __builtin_amdgcn_readfirstlane(t.q0);
  t.lq = __builtin_amdgcn_readfirstlane(t.lq);
  t.k0 = __builtin_amdgcn_readfirstlane(t.k0);
  t.lk = __builtin_amdgcn_readfirstlane(t.lk);
  t.block = __builtin_amdgcn_readfirstlane(t.block);
  t.live = __builtin_amdgcn_readfirstlane((int)t.live) != 0;
  return t;
}

}  // namespace naylis
