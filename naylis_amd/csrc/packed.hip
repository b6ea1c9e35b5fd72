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
#include "common.h"
#include "launch.h"
#include "packed_tiles.h"
#include "timing.h"

namespace naylis {

namespace {

constexpr int kStageRows = 64;

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
};

// Rows [row, row + rows) of one head, up to the sequence's end: a resource
// that reads zeros past it.  Built for each tile and stage from a 64-bit
// address, so that no sequence is too long for the 32-bit offsets within.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const bf16_t* base, long ld, int row, int len, int rows,
                                                            int hd) {
  const int live = min(len - row, rows);
  return make_rsrc(base + (long)row * ld, live > 0 ? ((uint32_t)(live - 1) * (uint32_t)ld + hd) * 2 : 0);
}

// A thread's share of a 64-row stage of one operand.
template <int HD>
struct StageCopy {
  static constexpr int N = kStageRows * HD / 8 / 256;  // 16-byte chunks
  int voff[N], lds[N];
  __device__ __forceinline__ StageCopy(int tid, int ld) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = (i * 256 + tid) / (HD / 8), c = tid % (HD / 8);
      voff[i] = (r * ld + c * 8) * 2;
      lds[i] = r * 2 * HD + ((c ^ swz<HD>(r)) << 4);
    }
  }
  __device__ __forceinline__ void load(uint4 (&x)[N], __amdgpu_buffer_rsrc_t rs) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      x[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rs, voff[i], 0, 0));
  }
  __device__ __forceinline__ void store(const uint4 (&x)[N], uint8_t* tile) const {
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<uint4*>(tile + lds[i]) = x[i];
  }
};

// B operand fragments of 32 rows straight from memory: lane l gets row l % 32
// of the resource, features 16 ks + 8 (l / 32) + e.
template <int HD>
__device__ __forceinline__ void load_rows(bf16x8 (&f)[HD / 16], __amdgpu_buffer_rsrc_t rs, int ld, int lane) {
  const int off = ((lane & 31) * ld + 8 * (lane >> 5)) * 2;
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks)
    f[ks] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rs, off + 32 * ks, 0, 0));
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

template <int N>
__device__ __forceinline__ void clear(f32x16 (&a)[N]) {
#pragma unroll
  for (int t = 0; t < N; ++t) a[t] = f32x16{};
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

// Forward: 4 waves of 32 queries.
template <int HD>
__global__ __launch_bounds__(256, HD == 64 ? 4 : 2) void packed_fwd_kernel(
    const bf16_t* __restrict__ q, const bf16_t* __restrict__ k, const bf16_t* __restrict__ v, bf16_t* __restrict__ o,
    float* __restrict__ lse, PackedSeqs s, PackedHeads d, float c) {
  constexpr int NT = HD / 32;
  __shared__ __align__(16) uint8_t kt[2][kStageRows * 2 * HD];
  __shared__ __align__(16) uint8_t vt[2][kStageRows * 2 * HD];
  const PackedTile tile = find_tile<false>(s, blockIdx.x / d.H);
  if (!tile.live) return;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Head hd(blockIdx.x % d.H, d);
  const bf16_t* qb = q + (long)tile.q0 * d.ldq + (long)hd.h * d.hsq;
  const bf16_t* kb = k + (long)tile.k0 * d.ldk + (long)hd.kvh * d.hsk;
  const bf16_t* vb = v + (long)tile.k0 * d.ldv + (long)hd.kvh * d.hsv;
  const int shift = tile.lk - tile.lq;  // query i sees keys up to i + shift
  const int q0 = tile.block * kTileRows + wave * 32, row = q0 + col;

  bf16x8 qf[HD / 16];
  load_rows<HD>(qf, rows_rsrc(qb, d.ldq, q0, tile.lq, 32, HD), (int)d.ldq, lane);
  const StageCopy<HD> ck(tid, (int)d.ldk), cv(tid, (int)d.ldv);
  const RowFrag<HD> rf(lane);
  const TransFrag<HD> tf(lane);
  f32x16 acc[NT];
  clear(acc);
  float m = kNegBig, l = 0.f;
  const int keys = min(tile.lq, (tile.block + 1) * kTileRows) + shift;  // seen by the tile's last query
  const int nst = (max(keys, 0) + kStageRows - 1) / kStageRows;
  uint4 xk[StageCopy<HD>::N], xv[StageCopy<HD>::N];
  ck.load(xk, rows_rsrc(kb, d.ldk, 0, tile.lk, kStageRows, HD));
  cv.load(xv, rows_rsrc(vb, d.ldv, 0, tile.lk, kStageRows, HD));
  ck.store(xk, kt[0]);
  cv.store(xv, vt[0]);
  lds_barrier();
  for (int st = 0; st < nst; ++st) {
    const int nx = min(st + 1, nst - 1) * kStageRows;  // past the last stage: loaded again, not read
    ck.load(xk, rows_rsrc(kb, d.ldk, nx, tile.lk, kStageRows, HD));
    cv.load(xv, rows_rsrc(vb, d.ldv, nx, tile.lk, kStageRows, HD));
    const uint8_t* ks_ = kt[st & 1];
    const uint8_t* vs_ = vt[st & 1];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      const int kv0 = st * kStageRows + 32 * sub;
      if (kv0 > q0 + 31 + shift) continue;  // above the diagonal (wave-uniform)
      f32x16 x = f32x16{};
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) x = mfma32(rf.get(ks_, 32 * sub, ks), qf[ks], x);
      if (kv0 + 31 > q0 + shift) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (kv0 + acc_row(g, i) > row + shift) x[i] = -INFINITY;
      }
      float mx = x[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
      if (__any(mx * c > m)) {
        // per query, so that a row's result does not depend on its neighbours'
        const float mr = xor32_f32(mx, [](float a, float b) { return fmaxf(a, b); }) * c;
        const float mn = fmaxf(m, mr);
        const float al = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= al;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[t][i] *= al;
      }
      float ls = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], c, -m));
        ls += x[i];
      }
      l += ls;
      const bf16x8 pf[2] = {pack8(x, 0), pack8(x, 8)};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] = mfma32(tf.get(vs_, 32 * sub + 16 * h, t), pf[h], acc[t]);
    }
    ck.store(xk, kt[(st + 1) & 1]);
    cv.store(xv, vt[(st + 1) & 1]);
    lds_barrier();
  }
  const float ls = xor32_f32(l, [](float a, float b) { return a + b; });
  if (row < tile.lq) {
    // a query without keys: zeros, and a log-sum-exp under which every backward weight is 0
    const bool none = row + shift < 0;
    const long at = (long)tile.q0 + row;
    store_row<HD>(o + (at * d.H + hd.h) * HD, acc, none ? 0.f : 1.f / ls, g);
    if (lse && g == 0) lse[(long)hd.h * s.T + at] = none ? INFINITY : m + log2f(ls);
  }
}

// dQ (and delta = rowsum(dO o), which the dK/dV kernel reads): the forward's
// walk with P from the log-sum-exp.
template <int HD>
__global__ __launch_bounds__(256, HD == 64 ? 3 : 2) void packed_bwd_dq_kernel(
    const bf16_t* __restrict__ q, const bf16_t* __restrict__ k, const bf16_t* __restrict__ v,
    const bf16_t* __restrict__ o, const float* __restrict__ lse, const bf16_t* __restrict__ dout,
    bf16_t* __restrict__ dq, float* __restrict__ delta, PackedSeqs s, PackedHeads d, float scale) {
  constexpr int NT = HD / 32;
  __shared__ __align__(16) uint8_t kt[2][kStageRows * 2 * HD];
  __shared__ __align__(16) uint8_t vt[2][kStageRows * 2 * HD];
  const PackedTile tile = find_tile<false>(s, blockIdx.x / d.H);
  if (!tile.live) return;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Head hd(blockIdx.x % d.H, d);
  const bf16_t* qb = q + (long)tile.q0 * d.ldq + (long)hd.h * d.hsq;
  const bf16_t* kb = k + (long)tile.k0 * d.ldk + (long)hd.kvh * d.hsk;
  const bf16_t* vb = v + (long)tile.k0 * d.ldv + (long)hd.kvh * d.hsv;
  const bf16_t* db = dout + (long)tile.q0 * d.ldd + (long)hd.h * d.hsd;
  const bf16_t* ob = o + ((long)tile.q0 * d.H + hd.h) * HD;
  const int shift = tile.lk - tile.lq;
  const int q0 = tile.block * kTileRows + wave * 32, row = q0 + col;
  const float c = scale * kLog2e;

  bf16x8 qf[HD / 16], df[HD / 16];
  load_rows<HD>(qf, rows_rsrc(qb, d.ldq, q0, tile.lq, 32, HD), (int)d.ldq, lane);
  load_rows<HD>(df, rows_rsrc(db, d.ldd, q0, tile.lq, 32, HD), (int)d.ldd, lane);
  const long stat = (long)hd.h * s.T + tile.q0 + min(row, tile.lq - 1);
  const float ml = -lse[stat];
  float md = 0.f;  // -delta of the lane's query
  {
    bf16x8 of[HD / 16];
    load_rows<HD>(of, rows_rsrc(ob, (long)d.H * HD, q0, tile.lq, 32, HD), d.H * HD, lane);
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e) md = fmaf(-(float)df[ks][e], (float)of[ks][e], md);
    md = xor32_f32(md, [](float a, float b) { return a + b; });
    if (g == 0 && row < tile.lq) delta[stat] = -md;
  }
  const StageCopy<HD> ck(tid, (int)d.ldk), cv(tid, (int)d.ldv);
  const RowFrag<HD> rf(lane);
  const TransFrag<HD> tf(lane);
  f32x16 acc[NT];
  clear(acc);
  const int keys = min(tile.lq, (tile.block + 1) * kTileRows) + shift;
  const int nst = (max(keys, 0) + kStageRows - 1) / kStageRows;
  uint4 xk[StageCopy<HD>::N], xv[StageCopy<HD>::N];
  ck.load(xk, rows_rsrc(kb, d.ldk, 0, tile.lk, kStageRows, HD));
  cv.load(xv, rows_rsrc(vb, d.ldv, 0, tile.lk, kStageRows, HD));
  ck.store(xk, kt[0]);
  cv.store(xv, vt[0]);
  lds_barrier();
  for (int st = 0; st < nst; ++st) {
    const int nx = min(st + 1, nst - 1) * kStageRows;
    ck.load(xk, rows_rsrc(kb, d.ldk, nx, tile.lk, kStageRows, HD));
    cv.load(xv, rows_rsrc(vb, d.ldv, nx, tile.lk, kStageRows, HD));
    const uint8_t* ks_ = kt[st & 1];
    const uint8_t* vs_ = vt[st & 1];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      const int kv0 = st * kStageRows + 32 * sub;
      if (kv0 > q0 + 31 + shift) continue;
      f32x16 x = f32x16{}, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] = md;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        x = mfma32(rf.get(ks_, 32 * sub, ks), qf[ks], x);
        dp = mfma32(rf.get(vs_, 32 * sub, ks), df[ks], dp);
      }
      if (kv0 + 31 > q0 + shift) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (kv0 + acc_row(g, i) > row + shift) x[i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], c, ml)) * dp[i];
      const bf16x8 sf[2] = {pack8(x, 0), pack8(x, 8)};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] = mfma32(tf.get(ks_, 32 * sub + 16 * h, t), sf[h], acc[t]);
    }
    ck.store(xk, kt[(st + 1) & 1]);
    cv.store(xv, vt[(st + 1) & 1]);
    lds_barrier();
  }
  if (row < tile.lq) store_row<HD>(dq + (((long)tile.q0 + row) * d.H + hd.h) * HD, acc, scale, g);
}

// dK, dV: 4 waves of 32 keys, whose K and V rows stay in registers; for each
// query head of the group, the queries from the diagonal to the end pass
// through LDS with their -lse / c and -delta, which start the accumulators of
// S and dP.  Queries past the sequence get -inf there, so their P is 0.
template <int HD>
__global__ __launch_bounds__(256, HD == 64 ? 2 : 1) void packed_bwd_dkdv_kernel(
    const bf16_t* __restrict__ q, const bf16_t* __restrict__ k, const bf16_t* __restrict__ v,
    const float* __restrict__ lse, const bf16_t* __restrict__ dout, const float* __restrict__ delta,
    bf16_t* __restrict__ dk, bf16_t* __restrict__ dv, PackedSeqs s, PackedHeads d, float scale) {
  constexpr int NT = HD / 32;
  __shared__ __align__(16) uint8_t qt[2][kStageRows * 2 * HD];
  __shared__ __align__(16) uint8_t dt[2][kStageRows * 2 * HD];
  __shared__ __align__(16) float rows[2][2][kStageRows];  // [buffer][-lse / c, -delta][query]
  const PackedTile tile = find_tile<true>(s, blockIdx.x / d.Hkv);
  if (!tile.live) return;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % d.Hkv, group = d.H / d.Hkv;
  const bf16_t* kb = k + (long)tile.k0 * d.ldk + (long)kvh * d.hsk;
  const bf16_t* vb = v + (long)tile.k0 * d.ldv + (long)kvh * d.hsv;
  const bf16_t* qb = q + (long)tile.q0 * d.ldq + (long)kvh * group * d.hsq;
  const bf16_t* db = dout + (long)tile.q0 * d.ldd + (long)kvh * group * d.hsd;
  const long sb = (long)kvh * group * s.T + tile.q0;
  const int shift = tile.lk - tile.lq;
  const int kv0 = tile.block * kTileRows + wave * 32, row = kv0 + col;
  const float c = scale * kLog2e, rc = 1.f / c;

  bf16x8 kf[HD / 16], vf[HD / 16];
  load_rows<HD>(kf, rows_rsrc(kb, d.ldk, kv0, tile.lk, 32, HD), (int)d.ldk, lane);
  load_rows<HD>(vf, rows_rsrc(vb, d.ldv, kv0, tile.lk, 32, HD), (int)d.ldv, lane);
  const StageCopy<HD> cq(tid, (int)d.ldq), cd(tid, (int)d.ldd);
  const RowFrag<HD> rf(lane);
  const TransFrag<HD> tf(lane);
  f32x16 ak[NT], av[NT];
  clear(ak);
  clear(av);
  const int first = max(tile.block * kTileRows - shift, 0);  // the first query that sees a key of the tile
  const int st0 = first / kStageRows;
  const int nst = max((tile.lq + kStageRows - 1) / kStageRows - st0, 0), steps = nst * group;
  // threads 0 .. 63 carry -lse / c, 64 .. 127 -delta of the stage's queries
  auto load_stat = [&](int head, int st) {
    const int r = st * kStageRows + (tid & 63);
    const long i = sb + (long)head * s.T + min(r, tile.lq - 1);
    if (tid < 64) return r < tile.lq ? -lse[i] * rc : -INFINITY;
    return tid < 128 && r < tile.lq ? -delta[i] : 0.f;
  };
  uint4 xq[StageCopy<HD>::N], xd[StageCopy<HD>::N];
  float xs = 0.f;
  auto load = [&](int head, int st) {
    cq.load(xq, rows_rsrc(qb + (long)head * d.hsq, d.ldq, st * kStageRows, tile.lq, kStageRows, HD));
    cd.load(xd, rows_rsrc(db + (long)head * d.hsd, d.ldd, st * kStageRows, tile.lq, kStageRows, HD));
    xs = load_stat(head, st);
  };
  auto store = [&](int buf) {
    cq.store(xq, qt[buf]);
    cd.store(xd, dt[buf]);
    if (tid < 128) rows[buf][tid >> 6][tid & 63] = xs;
  };
  int head = 0, st = st0;
  if (steps > 0) {
    load(head, st);
    store(0);
  }
  lds_barrier();
  for (int step = 0; step < steps; ++step) {
    const int buf = step & 1, cur = st;
    if (step + 1 < steps) {  // the next stage, or the next head's first (past the last: loaded again, not read)
      if (++st == st0 + nst) {
        st = st0;
        ++head;
      }
    }
    load(head, st);
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      const int q0 = cur * kStageRows + 32 * sub;
      if (kv0 > q0 + 31 + shift) continue;  // above the diagonal
      f32x16 x, dp;
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
        x = mfma32(rf.get(qt[buf], 32 * sub, ks), kf[ks], x);
        dp = mfma32(rf.get(dt[buf], 32 * sub, ks), vf[ks], dp);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = __builtin_amdgcn_exp2f(x[i] * c);
      if (kv0 + 31 > q0 + shift) {
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
          av[t] = mfma32(tf.get(dt[buf], 32 * sub + 16 * h, t), pf[h], av[t]);
          ak[t] = mfma32(tf.get(qt[buf], 32 * sub + 16 * h, t), sf[h], ak[t]);
        }
    }
    store(buf ^ 1);
    lds_barrier();
  }
  if (row < tile.lk) {
    const long at = (((long)tile.k0 + row) * d.Hkv + kvh) * HD;
    store_row<HD>(dk + at, ak, scale, g);
    store_row<HD>(dv + at, av, 1.f, g);
  }
}

// The grid has one workgroup per (tile, head).
bool packed_supported(long n, long T, long Tk, long H, long Hkv) {
  return n > 0 && H > 0 && Hkv > 0 && n < (1 << 20) && T < (1L << 30) && Tk < (1L << 30) &&
         packed_tiles(T, n) * H < (1L << 31) && packed_tiles(Tk, n) * Hkv < (1L << 31);
}

hipError_t launch_packed_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const PackedSeqs& s,
                             const PackedHeads& d, int hd, float scale, hipStream_t st) {
  const dim3 grid((unsigned)(packed_tiles(s.T, s.n) * d.H));
  auto run = [&](auto kernel) {
    NAYLIS_TIMED("packed_fwd", st,
                 hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, (const bf16_t*)q, (const bf16_t*)k,
                                    (const bf16_t*)v, (bf16_t*)o, lse, s, d, scale * kLog2e));
  };
  if (hd == 64)
    run(packed_fwd_kernel<64>);
  else
    run(packed_fwd_kernel<128>);
  return hipGetLastError();
}

hipError_t launch_packed_bwd(const void* q, const void* k, const void* v, const void* o, const float* lse,
                             const void* dout, void* dq, void* dk, void* dv, float* delta, const PackedSeqs& s,
                             const PackedHeads& d, int hd, float scale, hipStream_t st) {
  const dim3 gq((unsigned)(packed_tiles(s.T, s.n) * d.H)), gk((unsigned)(packed_tiles(s.Tk, s.n) * d.Hkv));
  auto run_dq = [&](auto kernel) {
    NAYLIS_TIMED("packed_bwd_dq", st,
                 hipLaunchKernelGGL(kernel, gq, dim3(256), 0, st, (const bf16_t*)q, (const bf16_t*)k,
                                    (const bf16_t*)v, (const bf16_t*)o, lse, (const bf16_t*)dout, (bf16_t*)dq, delta,
                                    s, d, scale));
    return hipGetLastError();
  };
  auto run_dkdv = [&](auto kernel) {
    NAYLIS_TIMED("packed_bwd_dkdv", st,
                 hipLaunchKernelGGL(kernel, gk, dim3(256), 0, st, (const bf16_t*)q, (const bf16_t*)k,
                                    (const bf16_t*)v, lse, (const bf16_t*)dout, delta, (bf16_t*)dk, (bf16_t*)dv, s, d,
                                    scale));
    return hipGetLastError();
  };
  if (s.T > 0) {
    const hipError_t e = hd == 64 ? run_dq(packed_bwd_dq_kernel<64>) : run_dq(packed_bwd_dq_kernel<128>);
    if (e != hipSuccess) return e;
  }
  if (s.Tk == 0) return hipSuccess;
  return hd == 64 ? run_dkdv(packed_bwd_dkdv_kernel<64>) : run_dkdv(packed_bwd_dkdv_kernel<128>);
}

}  // namespace naylis
