// Which tile of which packed sequence a workgroup takes (packed attention).
//
// Sequences are given by their offsets alone, which are on the device, so the
// grid has the most tiles that T rows in n sequences can have, and a workgroup's
// first wave finds its tile from the offsets: no plan to build, nothing to
// copy, no extra launch.
//
// Up to 22 sequences (a range a lane): tiles are ranked by their work, in levels
// of 128 rows of the other operand, longest first.  F(x) = number of tiles with
// more than x rows is a sum over the sequences (one wave reduction), so a binary
// search over x finds a rank's level and one scan over the sequences its tile,
// about 0.5 us of a workgroup's time.
//
// More sequences: in their order, sequence i from slot start / TILE + i on, which
// leaves room for its tiles; a slot's sequence is found by a search of 64 at a
// time, two loads for up to 4094.  15 sequences of up to 2000 tokens, 8 heads of
// 128, take 72 us ranked and 82 in order (forward), 30 level, 60 332 and 317; 128 of
// up to 64 tokens, 16 heads of 64, 25 and 18, 4096 6200 and 600.
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

constexpr int kRankedRanges = 24;  // most ranges (sequences and the two outer ones) whose tiles are ranked

// most tiles (ranked), or slots, of `tile` rows that `rows` rows in n sequences have, the two outer ranges included
inline long packed_tiles(long rows, long n, int tile = kTileRows) {
  return n + 2 <= kRankedRanges ? (rows + (tile - 1) * (n + 2)) / tile : rows / tile + n + 2;
}

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

// Tile `nth` of a range's tiles (query tiles from the last one on: longest first).
template <bool KEYS, int TILE>
__device__ __forceinline__ PackedTile tile_of(const PackedSpan& p, bool outer, int nth) {
  PackedTile tile{p.q0, p.lq, p.k0, p.lk, 0, false};
  if (outer) (KEYS ? tile.lq : tile.lk) = 0;
  const int all = ((KEYS ? tile.lk : tile.lq) + TILE - 1) / TILE;
  tile.block = KEYS ? nth : all - 1 - nth;
  tile.live = nth >= 0 && nth < all;
  return tile;
}

template <bool KEYS, int TILE>
__device__ __forceinline__ PackedTile search_ranked(const PackedSeqs& s, int rank) {
  const int lane = threadIdx.x & 63;
  const PackedSpan mine = packed_span(s, lane);
  const bool outer = lane == 0 || lane == s.n + 1;
  const auto total = [&](int x) {
    return __builtin_amdgcn_readfirstlane(wave_allsum_i32(tiles_over<KEYS, TILE>(mine, outer, x)));
  };
  if (rank >= total(-1)) return PackedTile{0, 0, 0, 0, 0, false};
  // the first level whose work no tile before `rank` lies under: F(128 lo) <= rank
  const int most = KEYS ? mine.lq : mine.lk;
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
  const int left = rank - total(x);
  const int over = tiles_over<KEYS, TILE>(mine, outer, x), here = tiles_over<KEYS, TILE>(mine, outer, above) - over;
  int sum = here;  // inclusive scan
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int t = __shfl_up(sum, o, 64);
    if (lane >= o) sum += t;
  }
  const unsigned long long past = __ballot(sum > left);
  if (!past) return PackedTile{0, 0, 0, 0, 0, false};
  const int src = __ffsll(past) - 1;
  const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, src); };
  return tile_of<KEYS, TILE>(PackedSpan{of(mine.q0), of(mine.lq), of(mine.k0), of(mine.lk)},
                             src == 0 || src == s.n + 1, of(over) + left - of(sum - here));
}

template <bool KEYS, int TILE>
__device__ __forceinline__ PackedTile search_slots(const PackedSeqs& s, int at) {
  const int lane = threadIdx.x & 63, rows = KEYS ? s.Tk : s.T;
  const int32_t* cu = KEYS ? s.cu_k : s.cu_q;
  const auto slot = [&](int i) { return (i == 0 ? 0 : min(max(cu[i - 1], 0), rows)) / TILE + i; };
  int lo = 0, ranges = s.n + 2;  // the last of these whose slot is no later (range 0 has slot 0)
  while (ranges > 1) {
    const int stride = (ranges + 63) / 64, i = lane * stride;
    const unsigned long long early = __ballot(i < ranges && slot(lo + min(i, ranges - 1)) <= at) | 1;
    const int skip = (63 - __clzll(early)) * stride;
    lo += skip;
    ranges = min(stride, ranges - skip);
  }
  return tile_of<KEYS, TILE>(packed_span(s, lo), lo == 0 || lo == s.n + 1, at - slot(lo));
}

// The workgroup's tile: searched by its first wave alone (the others' vector
// units would do the same 300 instructions for nothing).
template <bool KEYS, int TILE = kTileRows>
__device__ __forceinline__ PackedTile find_tile(const PackedSeqs& s, int rank) {
  __shared__ PackedTile found;
  if (threadIdx.x < 64) {
    const PackedTile t =
        s.n + 2 <= kRankedRanges ? search_ranked<KEYS, TILE>(s, rank) : search_slots<KEYS, TILE>(s, rank);
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
