// Causal attention over packed sequences of different lengths, with grouped
// heads:  o_i = sum_j softmax_j(scale q_i . k_j) v_j  over the keys
// j <= i + lk - lq of i's own sequence (the last query sees the last key; a
// query before the first key sees none, and its result is 0).
//
// q, o (T, H, hd) and k, v (Tk, Hkv, hd), heads of 64 or 128, any token and
// head strides for q, k, v and dO; query head h reads key head h / (H / Hkv).
// The reference has one length per batch and equal heads (model.py:279-345).
//
// Products run on v_mfma_f32_32x32x16_bf16 (fragment layouts in common.h).
// The forward and the dQ kernel form S^T = K Q^T: a lane owns one query, its
// softmax state is one register, and P^T / dS^T leave the accumulators as the
// B operand of the next product.  The dK/dV kernel forms S = Q K^T, where a
// lane owns one key, and walks the queries of all heads of its group, so that
// shared heads' gradients are summed in one workgroup in a fixed order, in
// fp32, with no atomics.  Probabilities and dS enter their products as bf16
// (at most half a step, 2^-9 of a value's binade); all sums are fp32.
//
// Bound by power, and by the softmax's vector work, which in the gradient kernels
// follows a wave's products instead of running beside them.  Over 16k tokens, with the
// products that each gradient kernel forms again counted, the forward runs at 1.0 to
// 1.1 PFLOP/s with 16 heads of 128 (a large matrix product at 1.14 for as long) and 0.88
// to 0.95 of 64, dQ at 1.15 to 1.25 and 1.0, dK/dV at 1.17 to 1.26 and 1.0, by card and
// clock; on tensors of zeros, which take less power, at 1.4 and 1.2, 1.65 and 1.5, 1.6
// and 1.45.  Nine sequences of 48 .. 3885 tokens, 16 heads of 64: 103 to 123 us forward,
// 405 to 433 with the gradients; four of 499 .. 4093, 32 / 8 heads of 128: 208 to 239 and
// 890 to 941.  The first loads of a tile and the last tiles' tail are a quarter of such
// batches.
#include "common.h"
#include "launch.h"
#include "packed_tiles.h"
#include "timing.h"

#include <algorithm>
#include <type_traits>

namespace naylis {

namespace {

constexpr int kStageRows = 64;
// The forward's reference stays until a score (log2 domain) passes it by more:
// weights reach 2^8, which costs fp32 sums and bf16 weights nothing, and few
// tiles rescale the sums (of 32 queries one has a new maximum in most tiles).
constexpr float kSlack = 8.f;
// Past this (log2 domain) the reference's own rounding is more than 2^16 in a
// weight, as a fused score - reference leaves it; there scores are rounded first.
constexpr float kFarScore = 268435456.f;
// Past this the log-sum-exp's rounding shows in the weights of the gradients
// (2^-12 at most up to here): such rows' weights are formed against it and divided by
// their sum.
constexpr float kFarLse = 4096.f;

// log2 of a weight against the log-sum-exp `lse` of far scores
__device__ __forceinline__ float far_exponent(float x, float c, float lse) {
#pragma clang fp contract(off)
  const float rounded = x * c;
  return fabsf(lse) > kFarScore ? rounded - lse : fmaf(x, c, -lse);
}

// LDS rows of HD bf16 without padding; 16-byte chunk c of row r sits in slot
// c ^ swz(r).  16 consecutive rows' chunk c then cover 256 bytes (row
// fragments), and so do 4 consecutive rows' 64-byte groups (transposing reads).
template <int HD>
__device__ __forceinline__ int swz(int r) {
  if constexpr (HD == 64) return ((r & 2) << 1) | ((r >> 2) & 1) | ((r >> 2) & 2);
  return ((r & 3) << 2) | ((r >> 2) & 3);
}

// Fragment of rows row0 .. row0 + 31 (row0 a multiple of 32): lane l gets
// X(row0 + l % 32, 16 ks + 8 (l / 32) + e).
template <int HD>
struct RowFrag {
  int off[HD / 16];
  __device__ __forceinline__ explicit RowFrag(int lane) {
    const int r = lane & 31, g = lane >> 5;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) off[ks] = r * 2 * HD + (((2 * ks + g) ^ swz<HD>(r)) << 4);
  }
  __device__ __forceinline__ bf16x8 get(const uint8_t* tile, int row0, int ks) const {
    return *reinterpret_cast<const bf16x8*>(tile + row0 * 2 * HD + off[ks]);
  }
  // to a buffer that lies `bit` bytes (a power of two past the tile) off
  __device__ __forceinline__ void move(int bit) {
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) off[ks] ^= bit;
  }
};

// A fragment of X^T, features 32 t .. 32 t + 31, over rows k0 .. k0 + 15 (k0
// a multiple of 16): lds_frag_T<true, true> of common.h on the swizzled rows.
template <int HD>
struct TransFrag {
  int lo[HD / 32], hi[HD / 32];
  __device__ __forceinline__ explicit TransFrag(int lane) {
    const int q = lane >> 4, j = lane & 15, g = q >> 1, mq = q & 1, c = j & 3;
    const int r0 = (j >> 2) + 4 * g, r1 = r0 + 8, ch = 2 * (c & 1) + mq, b = 8 * (c >> 1);
#pragma unroll
    for (int t = 0; t < HD / 32; ++t) {
      lo[t] = r0 * 2 * HD + (((4 * t + ch) ^ swz<HD>(r0)) << 4) + b;
      hi[t] = r1 * 2 * HD + (((4 * t + ch) ^ swz<HD>(r1)) << 4) + b;
    }
  }
  __device__ __forceinline__ bf16x8 get(const uint8_t* tile, int k0, int t) const {
    const v4i16 a = lds_read_tr16(reinterpret_cast<const bf16_t*>(tile + k0 * 2 * HD + lo[t]));
    const v4i16 b = lds_read_tr16(reinterpret_cast<const bf16_t*>(tile + k0 * 2 * HD + hi[t]));
    typedef short v8i16 __attribute__((ext_vector_type(8)));
    const v8i16 v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(bf16x8, v);
  }
  __device__ __forceinline__ void move(int bit) {
#pragma unroll
    for (int t = 0; t < HD / 32; ++t) {
      lo[t] ^= bit;
      hi[t] ^= bit;
    }
  }
};

// The same two with one offset each, the others from it by XOR where they are
// used: an instruction for each read, and 14 registers fewer (heads of 128).
struct LeanFrag {
  int rows, trans;
  __device__ __forceinline__ explicit LeanFrag(int lane) {
    rows = RowFrag<128>(lane).off[0];
    trans = TransFrag<128>(lane).lo[0];
  }
  // not computed ahead and kept
  __device__ __forceinline__ void renew() { asm volatile("" : "+v"(rows), "+v"(trans)); }
  __device__ __forceinline__ void move(int bit) {
    rows ^= bit;
    trans ^= bit;
  }
  __device__ __forceinline__ bf16x8 get(const uint8_t* tile, int row0, int ks) const {
    return *reinterpret_cast<const bf16x8*>(tile + row0 * 256 + (rows ^ (ks << 5)));
  }
  __device__ __forceinline__ bf16x8 get_t(const uint8_t* tile, int k0, int t) const {
    const int lo = trans ^ (t << 6);  // 8 rows on, the swizzle differs in one bit
    const v4i16 a = lds_read_tr16(reinterpret_cast<const bf16_t*>(tile + k0 * 256 + lo));
    const v4i16 b = lds_read_tr16(reinterpret_cast<const bf16_t*>(tile + k0 * 256 + (lo ^ 0x820)));
    typedef short v8i16 __attribute__((ext_vector_type(8)));
    const v8i16 v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(bf16x8, v);
  }
};
struct FullFrag : RowFrag<64>, TransFrag<64> {
  __device__ __forceinline__ explicit FullFrag(int lane) : RowFrag<64>(lane), TransFrag<64>(lane) {}
  __device__ __forceinline__ void renew() {}
  __device__ __forceinline__ void move(int bit) {
    RowFrag<64>::move(bit);
    TransFrag<64>::move(bit);
  }
  __device__ __forceinline__ bf16x8 get(const uint8_t* tile, int row0, int ks) const {
    return RowFrag<64>::get(tile, row0, ks);
  }
  __device__ __forceinline__ bf16x8 get_t(const uint8_t* tile, int k0, int t) const {
    return TransFrag<64>::get(tile, k0, t);
  }
};

// Rows [row, row + rows) of one head, up to the sequence's end: a resource
// that reads zeros past it.  Built for each tile and stage from a 64-bit
// address, so that no sequence is too long for the 32-bit offsets within.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const bf16_t* base, long ld, int row, int len, int rows,
                                                            int hd) {
  const int live = min(len - row, rows);
  return make_rsrc(base + (long)row * ld, live > 0 ? ((uint32_t)(live - 1) * (uint32_t)ld + hd) * 2 : 0);
}

// A wave's share of the stages of one operand, 64 rows each, from memory to LDS
// directly: 64 lanes x 16 bytes land in lane order, so the swizzle is on the
// source side.  Rows past the sequence are zeros; a stage past it loads nothing
// but counts as loads in flight.  The load is written in assembly because the
// compiler would wait for every such load before the next transposing LDS read;
// it has no register output, and the waits in wait_loads are those that its
// readers need.
typedef int i32x4 __attribute__((ext_vector_type(4)));
template <int HD>
struct StageLoad {
  static constexpr int N = kStageRows * 2 * HD / 1024 / 4;  // loads of a wave
  const bf16_t* base;
  long ld;
  int len, wave, voff;  // (pieces lie 16 or 32 rows apart, where the swizzle is the same)
  __device__ __forceinline__ StageLoad(const bf16_t* p, long ld_, int len_, int wave_, int lane)
      : base(p), ld(ld_), len(len_), wave(wave_) {
    const int at = wave * 1024 + lane * 16, r = at / (2 * HD), ch = at % (2 * HD) / 16;
    voff = (r * (int)ld + (ch ^ swz<HD>(r)) * 8) * 2;
  }
  __device__ __forceinline__ void load(uint32_t lds, int stage) const {
    const int row = stage * kStageRows, live = min(len - row, kStageRows);
    const uint64_t a = (uint64_t)(base + (long)row * ld);
    const uint32_t bytes = live > 0 ? ((uint32_t)(live - 1) * (uint32_t)ld + HD) * 2 : 0;
    const i32x4 rs{(int)(uint32_t)a, (int)((a >> 32) & 0xffff), (int)bytes, 0x00020000};
#pragma unroll
    for (int i = 0; i < N; ++i)
      asm volatile(
          "s_mov_b32 m0, %0\n\t"
          "s_nop 0\n\t"
          "buffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds + (i * 4 + wave) * 1024),
          "v"(voff), "s"(rs), "s"(i * (4096 / HD) * (int)ld)
          : "memory", "m0");
  }
};

// 64 floats p[first ..] of len (zeros past it) to LDS, 4 bytes a lane.
__device__ __forceinline__ void load_floats(const float* p, int len, int first, int lane, uint32_t lds) {
  const uint64_t a = (uint64_t)(p + first);
  const i32x4 rs{(int)(uint32_t)a, (int)((a >> 32) & 0xffff), max(len - first, 0) * 4, 0x00020000};
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dword %1, %2, 0 offen lds" ::"s"(lds),
      "v"(lane * 4), "s"(rs)
      : "memory", "m0");
}

// All but the newest n loads of every wave are in LDS, and what the waves have
// read from LDS so far may be overwritten.
template <int n>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(n) : "memory");
}

// max(m, x0 .. x15) of a product's results.  In assembly because fmaxf quiets
// NaN first, an instruction more for each; m has to come from an instruction
// that reads one of the results and that the compiler places, because it counts
// the wait states after a matrix instruction, and not for assembly.
__device__ __forceinline__ float max_of(float m, const f32x16& x) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3\n\t"
      "v_max3_f32 %0, %0, %4, %5\n\t"
      "v_max3_f32 %0, %0, %6, %7\n\t"
      "v_max3_f32 %0, %0, %8, %9\n\t"
      "v_max3_f32 %0, %0, %10, %11\n\t"
      "v_max3_f32 %0, %0, %12, %13\n\t"
      "v_max3_f32 %0, %0, %14, %15"
      : "=&v"(r)
      : "v"(m), "v"(x[2]), "v"(x[3]), "v"(x[4]), "v"(x[5]), "v"(x[6]), "v"(x[7]), "v"(x[8]), "v"(x[9]), "v"(x[10]),
        "v"(x[11]), "v"(x[12]), "v"(x[13]), "v"(x[14]), "v"(x[15]));
  return r;
}

// B operand fragments of 32 rows straight from memory: lane l gets row l % 32
// of the resource, features 16 ks + 8 (l / 32) + e.
template <int HD>
__device__ __forceinline__ void load_rows(bf16x8 (&f)[HD / 16], __amdgpu_buffer_rsrc_t rs, int ld, int lane) {
  const int off = ((lane & 31) * ld + 8 * (lane >> 5)) * 2;
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks)
    f[ks] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rs, off + 32 * ks, 0, 0));
}

// The fragments are here from now on.  Without this the compiler, which does not
// see wait_loads' waits, waits for them at every use, and so in every round for
// the stages under way (forward, 16k tokens, 16 heads of 128: 1055 -> 1032 us).
template <int N>
__device__ __forceinline__ void arrived(bf16x8 (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

// Order of a block of products whose operands come from LDS: N1 products of R1
// reads each, then N2 of R2; the reads of two products ahead of the products, and
// FIRST other reads before them.  Left alone the compiler reads each operand right
// before its product, into the registers of the last one, and waits there: dK/dV of
// four sequences of 499 .. 4093, 32 / 8 heads of 128, 488 -> 421 us, dQ 324 -> 317.
// Three products ahead: level.
template <int N1, int R1, int N2 = 0, int R2 = 0, int FIRST = 0>
__device__ __forceinline__ void read_ahead() {
  constexpr int MFMA = 0x8, DS_READ = 0x100;
  __builtin_amdgcn_sched_group_barrier(DS_READ, FIRST + 2 * R1, 0);
#pragma unroll
  for (int i = 0; i < N1 - 2; ++i) {
    __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
    __builtin_amdgcn_sched_group_barrier(DS_READ, R1, 0);
  }
#pragma unroll
  for (int i = 0; i < N2; ++i) {
    __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
    __builtin_amdgcn_sched_group_barrier(DS_READ, R2, 0);
  }
  __builtin_amdgcn_sched_group_barrier(MFMA, 2, 0);
}

// Transposed accumulators (lane = row, registers = features 32 t + 16 g + v)
// times x to a row of HD bf16.
template <int HD>
__device__ __forceinline__ void store_row(bf16_t* p, const f32x16 (&a)[HD / 32], float x, int g) {
#pragma unroll
  for (int t = 0; t < HD / 32; ++t) {
    f32x16 s;
#pragma unroll
    for (int v = 0; v < 16; ++v) s[v] = a[t][v] * x;
    *reinterpret_cast<bf16x8*>(p + 32 * t + 16 * g) = pack8(s, 0);
    *reinterpret_cast<bf16x8*>(p + 32 * t + 16 * g + 8) = pack8(s, 8);
  }
}

// The same to a row of HD fp32.
template <int HD>
__device__ __forceinline__ void store_row_f32(float* p, const f32x16 (&a)[HD / 32], float x, int g) {
#pragma unroll
  for (int t = 0; t < HD / 32; ++t)
#pragma unroll
    for (int v = 0; v < 16; v += 4)
      *reinterpret_cast<f32x4*>(p + 32 * t + 16 * g + v) =
          f32x4{a[t][v] * x, a[t][v + 1] * x, a[t][v + 2] * x, a[t][v + 3] * x};
}

// The same as two bf16 tensors: the rounded values, and what rounding left.
template <int HD>
__device__ __forceinline__ void store_row_hilo(bf16_t* p, bf16_t* rest, const f32x16 (&a)[HD / 32], float x, int g) {
#pragma unroll
  for (int t = 0; t < HD / 32; ++t) {
    f32x16 s;
#pragma unroll
    for (int v = 0; v < 16; ++v) s[v] = a[t][v] * x;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 hi, lo;
      pack8_hilo(s, 8 * h, hi, lo);
      *reinterpret_cast<bf16x8*>(p + 32 * t + 16 * g + 8 * h) = hi;
      *reinterpret_cast<bf16x8*>(rest + 32 * t + 16 * g + 8 * h) = lo;
    }
  }
}

template <int N>
__device__ __forceinline__ void clear(f32x16 (&a)[N]) {
#pragma unroll
  for (int t = 0; t < N; ++t) a[t] = f32x16{};
}

// N accumulators of the odd wave of a pair added to the even one's through LDS
// (`sums`: the pair's 64 N x 64 bytes), which the workgroup no longer needs
// otherwise, and so `one` where it is given (256 bytes more).  The odd wave's
// work ends here.
template <int N>
__device__ __forceinline__ void join_pair(f32x16 (&a)[N], uint8_t* sums, int share, int lane, float* one = nullptr) {
  f32x4* p = reinterpret_cast<f32x4*>(sums) + lane;
  lds_barrier();
  if (share == 1) {
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        p[(4 * t + i) * 64] = f32x4{a[t][4 * i], a[t][4 * i + 1], a[t][4 * i + 2], a[t][4 * i + 3]};
    if (one) reinterpret_cast<float*>(sums + N * 4096)[lane] = *one;
  }
  lds_barrier();
  if (share == 1) return;
  if (one) *one += reinterpret_cast<const float*>(sums + N * 4096)[lane];
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 b = p[(4 * t + i) * 64];
#pragma unroll
      for (int e = 0; e < 4; ++e) a[t][4 * i + e] += b[e];
    }
}

// Head of position hh: key heads innermost, so that the workgroups that an XCD
// gets (every eighth) share few key heads and keep them in its L2.
struct Head {
  int h, kvh;
  __device__ __forceinline__ Head(int hh, const PackedHeads& d) {
    kvh = hh % d.Hkv;
    h = kvh * (d.H / d.Hkv) + hh / d.Hkv;
  }
};

}  // namespace

// Forward: 4 waves of 32 queries.  The walk over 32-key tiles is pipelined by
// one: while the vector units take the exponentials of tile t, the matrix units
// form the scores of tile t + 1, and while those add P V of tile t, the maximum
// of tile t + 1 is found.  K and V stages go from memory to LDS directly, K a
// stage further ahead than V, each into the buffer that the barrier before has
// freed: barrier 1 of a stage stands after the last use of its K, barrier 2
// after that of its V.
// SPLIT 2, for grids that leave CUs idle: 64 queries, each 32 of them with two
// waves, which take the even and the odd key tiles (one of each stage, so that one
// barrier a stage does) and join their sums at the end.
template <int HD, int SPLIT>
__global__ __launch_bounds__(256, HD == 64 ? 3 : 2) void packed_fwd_kernel(
    const bf16_t* __restrict__ q, const bf16_t* __restrict__ k, const bf16_t* __restrict__ v, bf16_t* __restrict__ o,
    bf16_t* __restrict__ rest, float* __restrict__ lse, PackedSeqs s, PackedHeads d, float c) {
  constexpr int NT = HD / 32, NK = HD / 16, STAGE = kStageRows * 2 * HD, ROWS = kTileRows / SPLIT;
  __shared__ __align__(1024) uint8_t ring[4 * STAGE];  // K even, K odd, V even, V odd
  const PackedTile tile = find_tile<false, ROWS>(s, blockIdx.x / d.H);
  if (!tile.live) return;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Head hd(blockIdx.x % d.H, d);
  const bf16_t* qb = q + (long)tile.q0 * d.ldq + (long)hd.h * d.hsq;
  const int shift = tile.lk - tile.lq;  // query i sees keys up to i + shift
  const int q0 = tile.block * ROWS + wave / SPLIT * 32, row = q0 + col, share = wave % SPLIT;

  bf16x8 qf[NK];
  load_rows<HD>(qf, rows_rsrc(qb, d.ldq, q0, tile.lq, 32, HD), (int)d.ldq, lane);
  const StageLoad<HD> lk(k + (long)tile.k0 * d.ldk + (long)hd.kvh * d.hsk, d.ldk, tile.lk, wave, lane);
  const StageLoad<HD> lv(v + (long)tile.k0 * d.ldv + (long)hd.kvh * d.hsv, d.ldv, tile.lk, wave, lane);
  RowFrag<HD> rf(lane);
  TransFrag<HD> tf(lane);
  tf.move(2 * STAGE);
  const uint32_t ring0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)ring;  // LDS byte address
  const int keys = min(tile.lq, (tile.block + 1) * ROWS) + shift;  // seen by the tile's last query
  const int nst = (max(keys, 0) + kStageRows - 1) / kStageRows;
  // key tiles that the wave's queries see (a wave behind the sequence has none)
  const int nt = q0 < tile.lq ? min(max(q0 + 32 + shift + 31, 0) / 32, 2 * nst) : 0;

  f32x16 acc[NT], x;  // x: scores of the tile at hand
  clear(acc);
  float m = kLowest, l = 0.f, inf;
  float ce = c;      // what scores are multiplied by: 1 in lanes whose scores are far and were multiplied before
  bool far = false;  // whether the wave has such lanes
  // (a known infinity would turn the median below into a maximum of three instructions)
  asm("s_mov_b32 %0, 0x7f800000" : "=s"(inf));
  // mask of tile t, its maximum, and the sums rescaled where that is far above the reference
  auto settle = [&](f32x16& z, int t) {
    auto times_c = [&](bool mine) {
      const float f = mine ? c : 1.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) z[i] *= f;
    };
    if (32 * t + 31 > q0 + shift || far) {
      asm volatile("");  // a branch, not 16 selects for every tile
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (32 * t + acc_row(g, i) > row + shift) z[i] = -INFINITY;
      if (far) times_c(ce != c);
    }
    auto over_of = [&]() { return fmaf(max_of(__builtin_amdgcn_fmed3f(z[0], z[1], inf), z), ce, -kSlack); };
    const float over = over_of();
    if (__builtin_expect(__any(over > m), 0)) {
      // per query, so that a row's result does not depend on its neighbours'
      const auto fmx = [](float a, float b) { return fmaxf(a, b); };
      float most = xor32_f32(over, fmx);
      const bool turns = fabsf(most) > kFarScore && most != -INFINITY && ce == c;
      if (__any(turns)) {
        far = true;
        times_c(turns);
        if (turns) ce = 1.f;
        most = xor32_f32(over_of(), fmx);
      }
      const float mn = most > m ? most + kSlack : m;
      const float al = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= al;
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[u][i] *= al;
    }
  };
  auto weigh = [&](f32x16& p, int i) {
    p[i] = __builtin_amdgcn_exp2f(SPLIT == 1 ? p[i] : fmaf(p[i], ce, -m));
    l += p[i];
  };
  // Tile t (the first or second of its stage) with its scores in x; leaves those of
  // the wave's next one, t + SPLIT, there.  The lanes' LDS offsets move to the other
  // buffer a stage at a time, so that tiles differ by constants.
  auto step = [&](auto second, int t) {
    constexpr int HALF = 32 * 2 * HD, SECOND = decltype(second)::value;
    const uint8_t* vb = ring + SECOND * HALF;
    const uint8_t* kb = ring + (SECOND != (SPLIT == 1) ? HALF : 0);
    f32x16 p = x;  // weights; their exponents before the branch, so that the next scores can take x's registers
    if constexpr (SPLIT == 1) {
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = fmaf(x[i], ce, -m);
    }
    auto add_pv = [&]() {
      const bf16x8 pf[2] = {pack8(p, 0), pack8(p, 8)};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int u = 0; u < NT; ++u) acc[u] = mfma32(tf.get(vb, 16 * h, u), pf[h], acc[u]);
    };
    if (t + SPLIT < nt) {
      x = f32x16{};
#pragma unroll
      for (int ks = 0; ks < NK; ++ks) {
        x = mfma32(rf.get(kb, 0, ks), qf[ks], x);
#pragma unroll
        for (int i = 0; i < 16 / NK; ++i) weigh(p, ks * (16 / NK) + i);
      }
      add_pv();
      read_ahead<NK, 1, 2 * NT, 2>();
      settle(x, t + SPLIT);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) weigh(p, i);
      add_pv();
    }
  };

  lk.load(ring0, 0);
  lv.load(ring0 + 2 * STAGE, 0);
  lk.load(ring0 + STAGE, 1);
  arrived(qf);
  wait_loads<StageLoad<HD>::N>();
  if (share < nt) {
    x = f32x16{};
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) x = mfma32(rf.get(ring + share * 32 * 2 * HD, 0, ks), qf[ks], x);
    settle(x, share);
  }
  if constexpr (SPLIT == 1) {
    for (int st = 0; st < nst; ++st) {
      lv.load(ring0 + (2 + ((st + 1) & 1)) * STAGE, st + 1);
      if (2 * st < nt) step(std::false_type{}, 2 * st);
      wait_loads<StageLoad<HD>::N>();  // K of stage st + 1 is in LDS, that of st no longer needed
      lk.load(ring0 + (st & 1) * STAGE, st + 2);
      rf.move(STAGE);
      if (2 * st + 1 < nt) step(std::true_type{}, 2 * st + 1);
      wait_loads<StageLoad<HD>::N>();  // V likewise
      tf.move(STAGE);
    }
  } else {
    for (int st = 0; st < nst; ++st) {
      wait_loads<0>();  // K of stage st + 1 and V of st are in LDS, what stage st - 1 used is free
      rf.move(STAGE);
      lk.load(ring0 + (st & 1) * STAGE, st + 2);
      lv.load(ring0 + (2 + ((st + 1) & 1)) * STAGE, st + 1);
      if (2 * st + share < nt) {
        if (share)
          step(std::true_type{}, 2 * st + 1);
        else
          step(std::false_type{}, 2 * st);
      }
      tf.move(STAGE);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the late loads (zeros) land before LDS goes to another workgroup
  if constexpr (SPLIT == 2) {  // the odd tiles' sums to the even ones' (kLowest and zeros where there were none)
    float* sums = reinterpret_cast<float*>(ring) + wave / 2 * (HD / 2 + 2) * 64 + lane;
    lds_barrier();
    if (share == 1) {
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) sums[(16 * u + i) * 64] = acc[u][i];
      sums[HD / 2 * 64] = m;
      sums[(HD / 2 + 1) * 64] = l;
    }
    lds_barrier();
    if (share == 1) return;
    const float mo = sums[HD / 2 * 64], mn = fmaxf(m, mo);
    const float a = __builtin_amdgcn_exp2f(m - mn), b = __builtin_amdgcn_exp2f(mo - mn);
    m = mn;
    l = l * a + sums[(HD / 2 + 1) * 64] * b;
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[u][i] = acc[u][i] * a + sums[(16 * u + i) * 64] * b;
  }
  const float ls = xor32_f32(l, [](float a, float b) { return a + b; });
  if (row < tile.lq) {
    // a query without keys: zeros, and a log-sum-exp under which every backward weight is 0
    const bool none = row + shift < 0;
    if (none) clear(acc);  // (0 times a NaN of rows that its neighbours see)
    const long at = (long)tile.q0 + row;
    const long off = (at * d.H + hd.h) * HD;
    if (lse)
      store_row_hilo<HD>(o + off, rest + off, acc, none ? 0.f : 1.f / ls, g);
    else
      store_row<HD>(o + off, acc, none ? 0.f : 1.f / ls, g);
    if (lse && g == 0) lse[(long)hd.h * s.T + at] = none ? INFINITY : m + log2f(ls);
  }
}

// dQ: the forward's walk with P from the log-sum-exp.  Leaves (2, H, T) for the
// dK/dV kernel: -lse / c and -delta, delta = rowsum(dO o) of the forward's o
// before its rounding (o + rest): with the rounded o alone the error of dQ and dK
// (2-norm, against fp64) is 2.6e-3, with both 2.4e-3, of which each rounding that
// remains, of dS and of the result, makes 1.7e-3.  Rows of far scores leave -inf
// and log2 of the sum of their weights against the log-sum-exp.
// SPLIT as in the forward.
template <int HD, int SPLIT>
__global__ __launch_bounds__(256, HD == 64 ? 3 : 2) void packed_bwd_dq_kernel(
    const bf16_t* __restrict__ q, const bf16_t* __restrict__ k, const bf16_t* __restrict__ v,
    const bf16_t* __restrict__ o, const bf16_t* __restrict__ rest, const float* __restrict__ lse,
    const bf16_t* __restrict__ dout, bf16_t* __restrict__ dq, float* __restrict__ stats, PackedSeqs s, PackedHeads d,
    float scale) {
  constexpr int NT = HD / 32, STAGE = kStageRows * 2 * HD, ROWS = kTileRows / SPLIT;
  __shared__ __align__(1024) uint8_t ring[4 * STAGE];  // K even, K odd, V even, V odd
  const PackedTile tile = find_tile<false, ROWS>(s, blockIdx.x / d.H);
  if (!tile.live) return;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Head hd(blockIdx.x % d.H, d);
  const bf16_t* qb = q + (long)tile.q0 * d.ldq + (long)hd.h * d.hsq;
  const bf16_t* kb = k + (long)tile.k0 * d.ldk + (long)hd.kvh * d.hsk;
  const bf16_t* vb = v + (long)tile.k0 * d.ldv + (long)hd.kvh * d.hsv;
  const bf16_t* db = dout + (long)tile.q0 * d.ldd + (long)hd.h * d.hsd;
  const long ob = ((long)tile.q0 * d.H + hd.h) * HD;
  const int shift = tile.lk - tile.lq;
  const int q0 = tile.block * ROWS + wave / SPLIT * 32, row = q0 + col, share = wave % SPLIT;
  const float c = scale * kLog2e;

  bf16x8 qf[HD / 16], df[HD / 16];
  load_rows<HD>(qf, rows_rsrc(qb, d.ldq, q0, tile.lq, 32, HD), (int)d.ldq, lane);
  load_rows<HD>(df, rows_rsrc(db, d.ldd, q0, tile.lq, 32, HD), (int)d.ldd, lane);
  const long stat = (long)hd.h * s.T + tile.q0 + min(row, tile.lq - 1);
  const float ml = -lse[stat];
  float md = 0.f;  // -delta of the lane's query
  // per query, so that a row's gradient does not depend on its neighbours'
  const bool renew = ml != -INFINITY && !(fabsf(ml) <= fminf(kFarLse, 1e30f * c));
  const bool far = __any(renew);
  const float ce = renew && fabsf(ml) > kFarScore ? 1.f : c;  // (1: scores are multiplied and rounded first)
  float sum = 0.f;                                            // of a renewed row's weights
  {
    bf16x8 of[HD / 16], lf[HD / 16];
    load_rows<HD>(of, rows_rsrc(o + ob, (long)d.H * HD, q0, tile.lq, 32, HD), d.H * HD, lane);
    load_rows<HD>(lf, rows_rsrc(rest + ob, (long)d.H * HD, q0, tile.lq, 32, HD), d.H * HD, lane);
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e) md = fmaf(-(float)df[ks][e], (float)of[ks][e] + (float)lf[ks][e], md);
    md = xor32_f32(md, [](float a, float b) { return a + b; });
    if (g == 0 && share == 0 && row < tile.lq) {
      stats[stat] = renew ? -INFINITY : ml == -INFINITY ? 0.f : ml / c;  // (a row without keys is masked throughout)
      if (!renew) stats[(long)d.H * s.T + stat] = md;
    }
  }
  const StageLoad<HD> lk(kb, d.ldk, tile.lk, wave, lane), lv(vb, d.ldv, tile.lk, wave, lane);
  RowFrag<HD> rf(lane);
  TransFrag<HD> tf(lane);
  const uint32_t ring0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)ring;
  f32x16 acc[NT];
  clear(acc);
  const int keys = min(tile.lq, (tile.block + 1) * ROWS) + shift;
  const int nst = (max(keys, 0) + kStageRows - 1) / kStageRows;
  lk.load(ring0, 0);
  lv.load(ring0 + 2 * STAGE, 0);
  arrived(qf);
  arrived(df);
  for (int st = 0; st < nst; ++st) {
    wait_loads<0>();  // stage st is in LDS, st - 1 read by every wave
    lk.load(ring0 + ((st + 1) & 1) * STAGE, st + 1);
    lv.load(ring0 + (2 + ((st + 1) & 1)) * STAGE, st + 1);
#pragma unroll
    for (int i2 = 0; i2 < 2 / SPLIT; ++i2) {
      const int sub = SPLIT == 1 ? i2 : share, kv0 = st * kStageRows + 32 * sub;
      if (kv0 > q0 + 31 + shift || q0 >= tile.lq) continue;
      f32x16 x = f32x16{}, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] = md;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        x = mfma32(rf.get(ring, 32 * sub, ks), qf[ks], x);
        dp = mfma32(rf.get(ring + 2 * STAGE, 32 * sub, ks), df[ks], dp);
      }
      read_ahead<HD / 8, 1>();
      if (kv0 + 31 > q0 + shift || far) {
        asm volatile("");  // a branch, not 16 selects for every tile
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (kv0 + acc_row(g, i) > row + shift) x[i] = -INFINITY;
        if (far) {
          const float f = ce != c ? c : 1.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            x[i] *= f;
            sum += __builtin_amdgcn_exp2f(fmaf(x[i], ce, ml));
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], ce, ml)) * dp[i];
      const bf16x8 sf[2] = {pack8(x, 0), pack8(x, 8)};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] = mfma32(tf.get(ring, 32 * sub + 16 * h, t), sf[h], acc[t]);
      read_ahead<2 * NT, 2>();
    }
    rf.move(STAGE);
    tf.move(STAGE);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the late loads (zeros) land before LDS goes to another workgroup
  if constexpr (SPLIT == 2) {
    join_pair(acc, ring + wave / 2 * 2 * STAGE, share, lane, &sum);
    if (share == 1) return;
  }
  float by = scale;
  if (far) {
    sum = xor32_f32(sum, [](float a, float b) { return a + b; });
    if (renew) by /= sum;
    if (renew && g == 0 && row < tile.lq) stats[(long)d.H * s.T + stat] = log2f(sum);
  }
  if (row + shift < 0) clear(acc);  // as in the forward
  if (row < tile.lq) store_row<HD>(dq + (((long)tile.q0 + row) * d.H + hd.h) * HD, acc, by, g);
}

// What only add_far_rows reads, of the workgroup's sequence and first heads: in LDS,
// because the scalar registers are the main loop's.
struct FarOperands {
  const bf16_t *k, *v, *o, *rest;
  const float* lse;
  int ldk, ldv;
};
// The lane, in no register until then.
__device__ __forceinline__ int lane_again() {
  return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));
}
template <typename T>
__device__ __forceinline__ T* uniform(T* p) {
  const uint64_t a = (uint64_t)p;
  return (T*)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)a) |
              (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32)) << 32);
}

// The far rows (-inf in `starts`, and the log2 of their weights' sum a stage behind) of
// 32 queries of head `head`, whose Q and dO are in LDS at row 32 sub, added to 32 keys'
// dK and dV.  Scores from the same products as in dQ, so that they are the same bits
// there and here; K, V and what -delta needs are read from memory again, because the
// registers are the main loop's.
template <int HD, typename Frag>
__device__ __forceinline__ void add_far_rows(f32x16 (&ak)[HD / 32], f32x16 (&av)[HD / 32], const FarOperands& in,
                                             const Frag& fr, const uint8_t* ring, const float* starts,
                                             const bf16_t* dout, int head, int T, const PackedTile& tile,
                                             const PackedHeads& d, int q0, int sub, int kv0, float c, int lane) {
  constexpr int NT = HD / 32, STAGE = kStageRows * 2 * HD;
  const int col = lane & 31, g = lane >> 5, shift = tile.lk - tile.lq;
  if (!__any(starts[32 * sub + col] == -INFINITY)) return;
  const float big = uniform(in.lse)[(long)head * T + min(q0 + col, tile.lq - 1)];
  const int ldk = __builtin_amdgcn_readfirstlane(in.ldk), ldv = __builtin_amdgcn_readfirstlane(in.ldv), ldo = d.H * HD;
  const auto kr = rows_rsrc(uniform(in.k), ldk, kv0, tile.lk, 32, HD),
             vr = rows_rsrc(uniform(in.v), ldv, kv0, tile.lk, 32, HD),
             dr = rows_rsrc(dout, d.ldd, q0, tile.lq, 32, HD),
             outr = rows_rsrc(uniform(in.o) + head * HD, ldo, q0, tile.lq, 32, HD),
             restr = rows_rsrc(uniform(in.rest) + head * HD, ldo, q0, tile.lq, 32, HD);
  const auto piece = [&](__amdgpu_buffer_rsrc_t rs, int ld, int ks) {
    const int off = (col * ld + 8 * g) * 2 + 32 * ks;
    return __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
  };
  float md = 0.f;  // -delta of query col
#pragma unroll 2
  for (int ks = 0; ks < HD / 16; ++ks) {
    const bf16x8 df = piece(dr, (int)d.ldd, ks), of = piece(outr, ldo, ks), lf = piece(restr, ldo, ks);
#pragma unroll
    for (int e = 0; e < 8; ++e) md = fmaf(-(float)df[e], (float)of[e] + (float)lf[e], md);
  }
  md = xor32_f32(md, [](float a, float b) { return a + b; });
  f32x16 x = f32x16{}, dp = f32x16{};
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks) {
    x = mfma32(fr.get(ring, 32 * sub, ks), piece(kr, ldk, ks), x);
    dp = mfma32(fr.get(ring + 2 * STAGE, 32 * sub, ks), piece(vr, ldv, ks), dp);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = acc_row(g, i);
    const float z = far_exponent(x[i], c, __shfl(big, r, 64)) - starts[kStageRows + 32 * sub + r];
    const float delta = __shfl(md, r, 64);
    const bool none = starts[32 * sub + r] != -INFINITY || kv0 + col > q0 + r + shift;
    x[i] = none ? 0.f : __builtin_amdgcn_exp2f(z);
    dp[i] = none ? 0.f : x[i] * (dp[i] + delta);
  }
  const bf16x8 pf[2] = {pack8(x, 0), pack8(x, 8)}, sf[2] = {pack8(dp, 0), pack8(dp, 8)};
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      av[t] = mfma32(fr.get_t(ring + 2 * STAGE, 32 * sub + 16 * h, t), pf[h], av[t]);
      ak[t] = mfma32(fr.get_t(ring, 32 * sub + 16 * h, t), sf[h], ak[t]);
    }
}

// dK, dV: waves of 32 keys, whose K and V rows stay in registers; for each query
// head of the group, the queries from the diagonal to the end pass through LDS with
// their -lse / c and -delta, which start the accumulators of S and dP.  Queries past
// the sequence are zeros throughout: their P is 1, their dO and dS 0.  Eight waves
// on stages of 128 queries take longer than two workgroups of four (470 -> 510 us,
// before read_ahead, for four sequences of 499 .. 4093, 32 / 8 heads of 128).
// Rows of far scores, whose -lse / c is -inf, have no weight there; where a workgroup
// met some, it walks again for them (all rows far: 6 to 7 times as long).
// parts > 1, for grids that leave CUs idle: a workgroup walks a part of the
// group's heads and leaves fp32 sums (parts, Tk, Hkv, HD) for packed_sum_kernel.
template <int HD, int KB>
__global__ __launch_bounds__(256, HD == 64 ? 3 : 2) void packed_bwd_dkdv_kernel(
    const bf16_t* __restrict__ q, const bf16_t* __restrict__ k, const bf16_t* __restrict__ v,
    const bf16_t* __restrict__ o, const bf16_t* __restrict__ rest, const float* __restrict__ lse,
    const bf16_t* __restrict__ dout, const float* __restrict__ stats, bf16_t* __restrict__ dk,
    bf16_t* __restrict__ dv, float* __restrict__ part_k, float* __restrict__ part_v, int parts, PackedSeqs s,
    PackedHeads d, float scale) {
  constexpr int NT = HD / 32, STAGE = kStageRows * 2 * HD;
  __shared__ __align__(1024) uint8_t ring[4 * STAGE];      // Q even, Q odd, dO even, dO odd
  __shared__ __align__(1024) float rows[2][2][kStageRows];  // [buffer][-lse / c, -delta][query]
  __shared__ FarOperands far_operands;
  __shared__ bool any_far;
  constexpr int SPLIT = 128 / KB;  // waves that share 32 keys, each with a part of every stage's queries
  const PackedTile tile = find_tile<true, KB>(s, blockIdx.x / (d.Hkv * parts));
  if (!tile.live) return;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % d.Hkv, part = blockIdx.x / d.Hkv % parts, all = d.H / d.Hkv;
  const int head0 = all * part / parts, group = all * (part + 1) / parts - head0;  // this part's heads
  const int h0 = kvh * all + head0;
  const bf16_t* kb = k + (long)tile.k0 * d.ldk + (long)kvh * d.hsk;
  const bf16_t* vb = v + (long)tile.k0 * d.ldv + (long)kvh * d.hsv;
  const bf16_t* qb = q + (long)tile.q0 * d.ldq + (long)h0 * d.hsq;
  const bf16_t* db = dout + (long)tile.q0 * d.ldd + (long)h0 * d.hsd;
  const long sb = (long)h0 * s.T + tile.q0;
  if (tid == 0) {
    const long ob = ((long)tile.q0 * d.H + h0) * HD;
    far_operands = FarOperands{kb, vb, o + ob, rest + ob, lse + sb, (int)d.ldk, (int)d.ldv};
    any_far = false;
  }
  const int shift = tile.lk - tile.lq;
  const int kv0 = tile.block * KB + wave / SPLIT * 32, row = kv0 + col, share = wave % SPLIT;
  const float c = scale * kLog2e;

  bf16x8 kf[HD / 16], vf[HD / 16];
  load_rows<HD>(kf, rows_rsrc(kb, d.ldk, kv0, tile.lk, 32, HD), (int)d.ldk, lane);
  load_rows<HD>(vf, rows_rsrc(vb, d.ldv, kv0, tile.lk, 32, HD), (int)d.ldv, lane);
  std::conditional_t<HD == 64, FullFrag, LeanFrag> fr(lane);
  const uint32_t ring0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)ring;
  const uint32_t rows0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)rows;
  f32x16 ak[NT], av[NT];
  clear(ak);
  clear(av);
  const int first = max(tile.block * KB - shift, 0);  // the first query that sees a key of the tile
  const int st0 = first / kStageRows;
  const int nst = max((tile.lq + kStageRows - 1) / kStageRows - st0, 0), steps = nst * group;
  StageLoad<HD> lq(qb, d.ldq, tile.lq, wave, lane), ld(db, d.ldd, tile.lq, wave, lane);
  // whether there were rows of far scores, whose weights are 0 in the products below (the look at each tile's
  // rows takes 1 % with heads of 64, 2 with 128; one wave's for all 3, a walk over them at the end 6)
  unsigned long long far = 0;
  // stage st of head `head` into buffer buf; past the last head nothing
  auto load = [&](int head, int st, int buf) {
    lq.base = qb + (long)head * d.hsq;
    ld.base = db + (long)head * d.hsd;
    lq.len = ld.len = head < group ? tile.lq : 0;
    lq.load(ring0 + buf * STAGE, st);
    ld.load(ring0 + (2 + buf) * STAGE, st);
    if (wave < 2) load_floats(stats + (long)wave * d.H * s.T + sb + (long)head * s.T, lq.len, st * kStageRows, lane,
                              rows0 + (buf * 2 + wave) * kStageRows * 4);
  };
  int head = 0, st = st0;
  load(steps > 0 ? 0 : group, st, 0);
  arrived(kf);
  arrived(vf);
  for (int step = 0; step < steps; ++step) {
    const int buf = step & 1, cur = st;
    if (++st == st0 + nst) {  // the next stage, or the next head's first
      st = st0;
      ++head;
    }
    wait_loads<0>();  // this step's stage is in LDS, the one before read by every wave
    load(head, st, buf ^ 1);
#pragma unroll
    for (int i2 = 0; i2 < 2 / SPLIT; ++i2) {
      const int sub = SPLIT == 1 ? i2 : share, q0 = cur * kStageRows + 32 * sub;
      if (kv0 > q0 + 31 + shift || q0 >= tile.lq || kv0 >= tile.lk) continue;  // above the diagonal, or outside
      fr.renew();
      f32x16 x, dp;
      far |= __ballot(rows[buf][0][32 * sub + (lane_again() & 31)] == -INFINITY);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(&rows[buf][0][32 * sub + 8 * i + 4 * g]);
        const f32x4 b = *reinterpret_cast<const f32x4*>(&rows[buf][1][32 * sub + 8 * i + 4 * g]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[4 * i + e] = a[e];
          dp[4 * i + e] = b[e];
        }
      }
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        x = mfma32(fr.get(ring, 32 * sub, ks), kf[ks], x);
        dp = mfma32(fr.get(ring + 2 * STAGE, 32 * sub, ks), vf[ks], dp);
      }
      read_ahead<HD / 8, 1, 0, 0, 9>();
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = __builtin_amdgcn_exp2f(x[i] * c);
      if (kv0 + 31 > q0 + shift) {
        asm volatile("");  // a branch, not 16 selects for every tile
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (row > q0 + acc_row(g, i) + shift) x[i] = 0.f;
      }
      const bf16x8 pf[2] = {pack8(x, 0), pack8(x, 8)};
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] *= dp[i];
      const bf16x8 sf[2] = {pack8(x, 0), pack8(x, 8)};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          av[t] = mfma32(fr.get_t(ring + 2 * STAGE, 32 * sub + 16 * h, t), pf[h], av[t]);
          ak[t] = mfma32(fr.get_t(ring, 32 * sub + 16 * h, t), sf[h], ak[t]);
        }
      read_ahead<4 * NT, 2>();
    }
    fr.move(STAGE);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the late loads (zeros) land before LDS goes to another workgroup
  if (far) any_far = true;
  lds_barrier();
  if (__builtin_expect(any_far, 0)) {  // the walk again, for those rows alone
    head = 0;
    st = st0;
    load(0, st, steps & 1);
    for (int step = steps; step < 2 * steps; ++step) {
      const int buf = step & 1, cur = st, cur_head = head;
      if (++st == st0 + nst) {
        st = st0;
        ++head;
      }
      wait_loads<0>();
      load(head, st, buf ^ 1);
      for (int sub = SPLIT == 1 ? 0 : share; sub < 2; sub += SPLIT) {
        const int q0 = cur * kStageRows + 32 * sub;
        if (kv0 > q0 + 31 + shift || q0 >= tile.lq || kv0 >= tile.lk) continue;
        add_far_rows<HD>(ak, av, far_operands, fr, ring, &rows[buf][0][0], db + (long)cur_head * d.hsd, cur_head, s.T,
                         tile, d, q0, sub, kv0, c, lane_again());
      }
      fr.move(STAGE);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  if constexpr (SPLIT == 2) {  // in two steps of half the ring
    join_pair(ak, ring + wave / 2 * STAGE, share, lane);
    join_pair(av, ring + (2 + wave / 2) * STAGE, share, lane);
    if (share == 1) return;
  }
  if (row < tile.lk) {
    const long at = (((long)tile.k0 + row) * d.Hkv + kvh) * HD, p = (long)part * s.Tk * d.Hkv * HD + at;
    if (parts == 1) {
      store_row<HD>(dk + at, ak, scale, g);
      store_row<HD>(dv + at, av, 1.f, g);
    } else {
      store_row_f32<HD>(part_k + p, ak, scale, g);
      store_row_f32<HD>(part_v + p, av, 1.f, g);
    }
  }
}

// Sums of the parts in their order, rounded once: dk (blockIdx.y 0) and dv.
__global__ __launch_bounds__(256) void packed_sum_kernel(const float* __restrict__ part_k,
                                                         const float* __restrict__ part_v, bf16_t* __restrict__ dk,
                                                         bf16_t* __restrict__ dv, long n, int parts) {
  const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const float* p = (blockIdx.y ? part_v : part_k) + i;
  f32x4 a = *reinterpret_cast<const f32x4*>(p);
  for (int k = 1; k < parts; ++k) a += *reinterpret_cast<const f32x4*>(p + k * n);
  bf16x4 o;
#pragma unroll
  for (int v = 0; v < 4; ++v) o[v] = (__bf16)a[v];
  *reinterpret_cast<bf16x4*>((blockIdx.y ? dv : dk) + i) = o;
}

// The grid has one workgroup per (tile, head), and a launch under 2^32 threads.
bool packed_supported(long n, long T, long Tk, long H, long Hkv) {
  return n > 0 && H > 0 && Hkv > 0 && n < (1 << 20) && T < (1L << 30) && Tk < (1L << 30) &&
         packed_tiles(T, n, 64) * H < (1L << 24) && packed_tiles(Tk, n, 64) * Hkv < (1L << 24);
}

// Two waves for 32 queries where the grid is under three quarters of the
// workgroups that run at once (two a CU with heads of 128, three of 64).
// Forward / dQ, us: 4000 queries of 8 heads of 128 92 -> 75 / 102 -> 78, 500 17 -> 14
// / 20 -> 17, of 16 heads of 64 75 -> 56 / 72 -> 65; beyond it 10 x 500 queries of 8
// heads of 128 20 -> 25 / 23 -> 33, 4000 of 32 150 -> 189 / 197 -> 220, of 24 heads
// of 64 82 -> 87 / 88 -> 93.
static bool packed_split(const PackedSeqs& s, const PackedHeads& d, int hd) {
  return packed_tiles(s.T, s.n) * d.H < (hd == 64 ? 576 : 384);
}

hipError_t launch_packed_fwd(const void* q, const void* k, const void* v, void* o, void* rest, float* lse,
                             const PackedSeqs& s, const PackedHeads& d, int hd, float scale, hipStream_t st) {
  auto run = [&](auto kernel, int rows) {
    NAYLIS_TIMED("packed_fwd", st,
                 hipLaunchKernelGGL(kernel, dim3((unsigned)(packed_tiles(s.T, s.n, rows) * d.H)), dim3(256), 0, st,
                                    (const bf16_t*)q, (const bf16_t*)k, (const bf16_t*)v, (bf16_t*)o, (bf16_t*)rest,
                                    lse, s, d, scale * kLog2e));
    return hipGetLastError();
  };
  const bool split = packed_split(s, d, hd);
  if (hd == 64) return split ? run(packed_fwd_kernel<64, 2>, 64) : run(packed_fwd_kernel<64, 1>, 128);
  return split ? run(packed_fwd_kernel<128, 2>, 64) : run(packed_fwd_kernel<128, 1>, 128);
}

// Tiles of 64 keys, whose waves share 32 of them, where those of 128 are under three
// a CU: 4000 tokens, 16 heads of 64, 88 -> 73 us; beyond it the join and the barriers
// cost more (nine sequences of 16376, 16 heads of 64, 189 -> 229; 8 x 2048, 16 heads of
// 128, 263 -> 322; 4000, 32 of 128, 233 -> 261).
static int packed_key_tile(const PackedSeqs& s, const PackedHeads& d) {
  return packed_tiles(s.Tk, s.n) * d.Hkv < 768 ? 64 : 128;
}

// Parts of a group where its key tiles are few, up to 1536 workgroups: 2000 tokens,
// 8 / 2 heads of 128 179 -> 55 us (and 4 for the sum), of 64 97 -> 33; 4000 tokens,
// 32 / 8 heads of 128 393 -> 284 (12).  With up to 2304 packed batches of 8192
// tokens take 309 us (and 25) for 293.  Not for short sequences, whose tiles have
// little to do (8 of 30 .. 128 tokens 12 -> 19 us).
static int packed_parts(const PackedSeqs& s, const PackedHeads& d, int hd) {
  const long wgs = std::max(packed_tiles(s.Tk, s.n, packed_key_tile(s, d)) * d.Hkv, 1L);
  if (s.T < 192L * s.n) return 1;
  return (int)std::max(1L, std::min((long)d.H / d.Hkv, 1536 / wgs));
}

size_t packed_bwd_ws_bytes(const PackedSeqs& s, const PackedHeads& d, int hd) {
  const int parts = packed_parts(s, d, hd);
  const size_t stats = (size_t)2 * d.H * s.T * 4;
  return (stats + 15) / 16 * 16 + (parts == 1 ? 0 : (size_t)2 * parts * s.Tk * d.Hkv * hd * 4);
}

hipError_t launch_packed_bwd(const void* q, const void* k, const void* v, const void* o, const void* rest,
                             const float* lse, const void* dout, void* dq, void* dk, void* dv, void* ws,
                             const PackedSeqs& s, const PackedHeads& d, int hd, float scale, hipStream_t st) {
  const int parts = packed_parts(s, d, hd);
  const long n = (long)s.Tk * d.Hkv * hd;  // elements of dk
  float* stats = (float*)ws;
  float* part_k = stats + ((size_t)2 * d.H * s.T + 3) / 4 * 4;
  float* part_v = part_k + parts * n;
  auto run_dq = [&](auto kernel, int rows) {
    NAYLIS_TIMED("packed_bwd_dq", st,
                 hipLaunchKernelGGL(kernel, dim3((unsigned)(packed_tiles(s.T, s.n, rows) * d.H)), dim3(256), 0, st,
                                    (const bf16_t*)q, (const bf16_t*)k, (const bf16_t*)v, (const bf16_t*)o,
                                    (const bf16_t*)rest, lse, (const bf16_t*)dout, (bf16_t*)dq, stats, s, d, scale));
    return hipGetLastError();
  };
  auto run_dkdv = [&](auto kernel, int rows) {
    NAYLIS_TIMED("packed_bwd_dkdv", st,
                 hipLaunchKernelGGL(kernel, dim3((unsigned)(packed_tiles(s.Tk, s.n, rows) * d.Hkv * parts)),
                                    dim3(256), 0, st, (const bf16_t*)q, (const bf16_t*)k, (const bf16_t*)v,
                                    (const bf16_t*)o, (const bf16_t*)rest, lse, (const bf16_t*)dout,
                                    (const float*)stats, (bf16_t*)dk, (bf16_t*)dv, part_k, part_v, parts, s, d,
                                    scale));
    return hipGetLastError();
  };
  if (s.T > 0) {
    const bool split = packed_split(s, d, hd);
    const hipError_t e = hd == 64 ? (split ? run_dq(packed_bwd_dq_kernel<64, 2>, 64)
                                           : run_dq(packed_bwd_dq_kernel<64, 1>, 128))
                                  : (split ? run_dq(packed_bwd_dq_kernel<128, 2>, 64)
                                           : run_dq(packed_bwd_dq_kernel<128, 1>, 128));
    if (e != hipSuccess) return e;
  }
  if (s.Tk == 0) return hipSuccess;
  const bool wide = packed_key_tile(s, d) == 128;
  const hipError_t e = hd == 64 ? (wide ? run_dkdv(packed_bwd_dkdv_kernel<64, 128>, 128)
                                        : run_dkdv(packed_bwd_dkdv_kernel<64, 64>, 64))
                                : (wide ? run_dkdv(packed_bwd_dkdv_kernel<128, 128>, 128)
                                        : run_dkdv(packed_bwd_dkdv_kernel<128, 64>, 64));
  if (e != hipSuccess || parts == 1) return e;
  NAYLIS_TIMED("packed_sum", st,
               hipLaunchKernelGGL(packed_sum_kernel, dim3((unsigned)((n / 4 + 255) / 256), 2), dim3(256), 0, st,
                                  (const float*)part_k, (const float*)part_v, (bf16_t*)dk, (bf16_t*)dv, n, parts));
  return hipGetLastError();
}

}  // namespace naylis
