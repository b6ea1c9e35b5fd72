// Packed attention, the paged cache, token log probabilities and the drafts'
// verification: argument checks, the C-ABI calls and the autograd nodes behind
// mom_kernels/hip_packed.py, hip_paged.py, hip_logprobs.py and hip_verify.py.  Calls without
// a gradient make no node; the checks are here, not in Python, because a call
// for one token costs little more than its host time.
#include "torch_common.h"

#include <cmath>

namespace naylis_ext {

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

namespace {

at::TensorOptions f32_like(const at::Tensor& t) { return t.options().dtype(at::kFloat); }

bool wants_grad(std::initializer_list<at::Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// Dual tensors need no requires_grad: a call that looked at that alone would
// return a constant for them.
void no_tangents(std::initializer_list<at::Tensor> ts, const char* who) {
  for (const at::Tensor& t : ts)
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), who, ": the forward-mode derivative is not implemented");
}

void on_gpu(const at::Tensor& t, const char* who, const char* name) {
  TORCH_CHECK(t.is_cuda(), who, ": ", name, " must be on a ROCm device, got ", t.device());
}

void same_device(const at::Tensor& t, const at::Tensor& q, const char* who, const char* name) {
  TORCH_CHECK(t.device() == q.device(), who, ": ", name, " is on ", t.device(), ", not on ", q.device());
}

// int32 and dense on q's device
at::Tensor indices(const at::Tensor& t, const at::Tensor& q, const char* who, const char* name) {
  same_device(t, q, who, name);
  TORCH_CHECK(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, who, ": ", name,
              " must be int32 or int64, got ", t.scalar_type());
  // int64 beyond int32 stays out of range instead of wrapping into it
  if (t.scalar_type() == at::kLong) return t.clamp(INT32_MIN, INT32_MAX).to(at::kInt).contiguous();
  return t.contiguous();
}

// Stream of a call: 0 is the current one, looked up here because that costs the
// caller in Python a tenth of a call for one token.
void* stream_of(int64_t st, const at::Tensor& t) { return st ? stream_ptr(st) : current_stream(t); }

double scale_of(const c10::optional<double>& scale, int64_t hd) { return scale ? *scale : 1.0 / std::sqrt((double)hd); }

// Strides of a (rows, heads, hd) operand; of a single row or head torch keeps any.
int64_t head_stride(const at::Tensor& t) { return t.size(1) == 1 ? t.size(2) : t.stride(1); }
int64_t row_stride(const at::Tensor& t) { return t.size(0) == 1 ? t.size(1) * t.size(2) : t.stride(0); }

// A (rows, heads, hd) operand as the kernels read it: whole 16-byte pieces at
// aligned addresses, features dense.  Anything else is copied.
at::Tensor rows_of(const at::Tensor& t) {
  const bool fits = t.stride(2) == 1 && row_stride(t) % 8 == 0 && head_stride(t) % 8 == 0 &&
                    row_stride(t) < (1 << 23) && (uintptr_t)t.data_ptr() % 16 == 0;
  if (fits) return t;
  const at::Tensor c = t.contiguous();
  return (uintptr_t)c.data_ptr() % 16 == 0 ? c : c.clone();
}

// ---- packed attention -----------------------------------------------------------

struct PackedArgs {
  at::Tensor q, k, v, cu_q, cu_k;
  double scale;
  int64_t n() const { return cu_q.size(0) - 1; }
};

// What a backward needs beside the inputs and the result.
struct PackedSaved {
  at::Tensor rest, lse;
};

at::Tensor packed_forward(const PackedArgs& a, PackedSaved* saved, void* st) {
  const int64_t T = a.q.size(0), Tk = a.k.size(0), H = a.q.size(1), hd = a.q.size(2);
  at::Tensor out = at::empty({T, H, hd}, a.q.options());
  const int64_t strides[6] = {row_stride(a.q), head_stride(a.q), row_stride(a.k),
                              head_stride(a.k), row_stride(a.v), head_stride(a.v)};
  if (saved) *saved = {at::empty_like(out), at::empty({H, T}, f32_like(a.q))};
  check(naylis_mom_packed_attn_fwd(a.q.data_ptr(), a.k.data_ptr(), a.v.data_ptr(), a.cu_q.data_ptr<int32_t>(),
                                   a.cu_k.data_ptr<int32_t>(), out.data_ptr(),
                                   saved ? saved->rest.data_ptr() : nullptr,
                                   saved ? saved->lse.data_ptr<float>() : nullptr, strides, (float)a.scale, a.n(), T,
                                   Tk, H, a.k.size(1), hd, st));
  return out;
}

variable_list packed_grads(const PackedArgs& a, const at::Tensor& out, const PackedSaved& saved,
                           const at::Tensor& grad) {
  at::DeviceGuard guard(a.q.device());
  const at::Tensor dout = rows_of(grad.to(a.q.scalar_type()));
  const int64_t T = a.q.size(0), Tk = a.k.size(0), H = a.q.size(1), Hkv = a.k.size(1), hd = a.q.size(2);
  at::Tensor dq = at::empty({T, H, hd}, a.q.options()), dk = at::empty({Tk, Hkv, hd}, a.q.options());
  at::Tensor dv = at::empty({Tk, Hkv, hd}, a.q.options());
  at::Tensor ws = workspace(need(naylis_mom_packed_attn_bwd_workspace_bytes(a.n(), T, Tk, H, Hkv, hd)), a.q);
  const int64_t strides[8] = {row_stride(a.q), head_stride(a.q), row_stride(a.k), head_stride(a.k),
                              row_stride(a.v), head_stride(a.v), row_stride(dout), head_stride(dout)};
  check(naylis_mom_packed_attn_bwd(a.q.data_ptr(), a.k.data_ptr(), a.v.data_ptr(), a.cu_q.data_ptr<int32_t>(),
                                   a.cu_k.data_ptr<int32_t>(), out.data_ptr(), saved.rest.data_ptr(),
                                   saved.lse.data_ptr<float>(), dout.data_ptr(),
                                   dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), ws.numel(), strides,
                                   (float)a.scale, a.n(), T, Tk, H, Hkv, hd, current_stream(a.q)));
  return {dq, dk, dv};
}

// The gradients as a node of their own, for a backward with create_graph: a
// second derivative raises instead of leaving this part out.
struct PackedAttentionGrad : public Function<PackedAttentionGrad> {
  static variable_list forward(AutogradContext*, at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor cu_q,
                               at::Tensor cu_k, at::Tensor out, at::Tensor rest, at::Tensor lse, at::Tensor dout,
                               double scale) {
    return packed_grads({q, k, v, cu_q, cu_k, scale}, out, {rest, lse}, dout);
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "packed_attention: the derivative of its backward is not implemented");
  }
};

struct PackedAttention : public Function<PackedAttention> {
  static at::Tensor forward(AutogradContext* ctx, at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor cu_q,
                            at::Tensor cu_k, double scale, int64_t st) {
    const PackedArgs a{rows_of(q), rows_of(k), rows_of(v), cu_q, cu_k, scale};
    PackedSaved saved;
    at::Tensor out = packed_forward(a, &saved, stream_ptr(st));
    ctx->save_for_backward({a.q, a.k, a.v, cu_q, cu_k, out, saved.rest, saved.lse});
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const double scale = ctx->saved_data["scale"].toDouble();
    variable_list g = at::GradMode::is_enabled()
                          ? PackedAttentionGrad::apply(s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], grads[0], scale)
                          : packed_grads({s[0], s[1], s[2], s[3], s[4], scale}, s[5], {s[6], s[7]}, grads[0]);
    g.resize(7);
    return g;
  }
};

at::Tensor packed_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& cu_q,
                            const at::Tensor& cu_k, c10::optional<double> scale_in, int64_t stream) {
  const char* who = "packed_attention";
  on_gpu(q, who, "q");
  at::DeviceGuard guard(q.device());
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && k.sizes() == v.sizes() && q.size(2) == k.size(2) && k.size(1) > 0 &&
                  q.size(1) > 0 && q.size(1) % k.size(1) == 0,
              who, ": needs q (T, H, hd) and k, v (Tk, Hkv, hd) with H a multiple of Hkv; got ", q.sizes(), ", ",
              k.sizes(), ", ", v.sizes());
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 && k.scalar_type() == at::kBFloat16 && v.scalar_type() == at::kBFloat16,
              who, ": q, k and v must be bf16");
  TORCH_CHECK(q.size(2) == 64 || q.size(2) == 128, who, ": head_dim ", q.size(2), " must be 64 or 128");
  same_device(k, q, who, "k");
  same_device(v, q, who, "v");
  const at::Tensor cq = indices(cu_q, q, who, "cu_seqlens");
  const at::Tensor ck = cu_k.is_same(cu_q) ? cq : indices(cu_k, q, who, "cu_seqlens_k");
  TORCH_CHECK(cq.dim() == 1 && cq.size(0) >= 2 && ck.sizes() == cq.sizes(), who,
              ": cu_seqlens and cu_seqlens_k must hold n + 1 offsets of the same n >= 1 sequences");
  no_tangents({q, k, v}, who);
  const double scale = scale_of(scale_in, q.size(2));
  void* st = stream_of(stream, q);
  if (wants_grad({q, k, v})) return PackedAttention::apply(q, k, v, cq, ck, scale, reinterpret_cast<int64_t>(st));
  at::NoGradGuard no_grad;
  return packed_forward({rows_of(q), rows_of(k), rows_of(v), cq, ck, scale}, nullptr, st);
}

// ---- paged cache ----------------------------------------------------------------

constexpr int kE4M3 = 2, kE2M1 = 3;

struct Cache {
  at::Tensor k, v, ks, vs;
  int dtype;
  int64_t pages, Hkv, page, hd;
  void* k_scale() const { return ptr(ks); }
  void* v_scale() const { return ptr(vs); }
};

// The pages are written in place and read where they are, so they have to be dense.
Cache cache_of(const at::Tensor& k, const at::Tensor& v, const c10::optional<at::Tensor>& ks,
               const c10::optional<at::Tensor>& vs, const char* who) {
  on_gpu(k, who, "the cache");
  TORCH_CHECK(k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() &&
                  v.device() == k.device() && k.is_contiguous() && v.is_contiguous() &&
                  (uintptr_t)k.data_ptr() % 16 == 0 && (uintptr_t)v.data_ptr() % 16 == 0,
              who, ": the cache's k and v must be dense (pages, Hkv, page_size, head_dim) tensors of one type and ",
              "device, 16-byte aligned; got ", k.sizes(), " ", k.scalar_type(), ", ", v.sizes(), " ", v.scalar_type());
  const bool codes = k.scalar_type() == at::kByte;
  TORCH_CHECK(codes || k.scalar_type() == at::kBFloat16, who,
              ": the cache must be bf16, or e4m3 or e2m1 codes in uint8 with scales; got ", k.scalar_type());
  TORCH_CHECK(codes == ks.has_value() && codes == vs.has_value(), who,
              ": e4m3 and e2m1 pages need k_scale and v_scale, bf16 pages have none");
  // the scales tell e2m1, two codes in a byte and an exponent's byte for 32, from e4m3
  const bool fp4 = codes && ks->scalar_type() == at::kByte;
  Cache c{k, v, ks.value_or(at::Tensor()), vs.value_or(at::Tensor()), fp4 ? kE2M1 : codes ? kE4M3 : kBF16,
          k.size(0), k.size(1), k.size(2), fp4 ? 2 * k.size(3) : k.size(3)};
  if (codes) {
    std::vector<int64_t> shape = k.sizes().slice(0, 3).vec();
    if (fp4) shape.push_back(c.hd / 32);
    for (const at::Tensor& s : {c.ks, c.vs})
      TORCH_CHECK(s.scalar_type() == c.ks.scalar_type() && (fp4 || s.scalar_type() == at::kFloat) &&
                      s.is_contiguous() && s.device() == k.device() && s.sizes() == shape &&
                      (uintptr_t)s.data_ptr() % 16 == 0,
                  who, ": k_scale and v_scale must be dense fp32 (pages, Hkv, page_size) tensors, or uint8 (pages, ",
                  "Hkv, page_size, head_dim / 32) ones for e2m1 pages, 16-byte aligned");
  }
  return c;
}

void written(const at::Tensor& t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// What an append is given beside the cache, checked and as the kernels read it.
struct NewTokens {
  at::Tensor k, v, table, pos, row;
  int64_t T;
  NewTokens(const Cache& c, const at::Tensor& k_in, const at::Tensor& v_in, const at::Tensor& table_in,
            const at::Tensor& positions, const c10::optional<at::Tensor>& rows, const char* who) {
    TORCH_CHECK(k_in.dim() == 3 && v_in.sizes() == k_in.sizes() && k_in.size(1) == c.Hkv && k_in.size(2) == c.hd &&
                    k_in.scalar_type() == at::kBFloat16 && v_in.scalar_type() == at::kBFloat16,
                who, ": k and v must be bf16 (T, Hkv, head_dim) of the cache's heads; got ", k_in.sizes(), " ",
                k_in.scalar_type(), ", ", v_in.sizes(), " ", v_in.scalar_type());
    same_device(k_in, c.k, who, "k");
    same_device(v_in, c.k, who, "v");
    table = indices(table_in, c.k, who, "block_table");
    pos = indices(positions, c.k, who, "positions");
    if (rows.has_value()) row = indices(*rows, c.k, who, "rows");
    T = k_in.size(0);
    TORCH_CHECK(table.dim() == 2 && table.size(1) > 0, who, ": block_table must be (B, pages of a sequence)");
    TORCH_CHECK(pos.dim() == 1 && pos.size(0) == T && (!row.defined() || row.sizes() == pos.sizes()), who,
                ": positions and rows must hold one entry for each of the ", T, " tokens");
    k = rows_of(k_in);
    v = rows_of(v_in);
  }
  const int32_t* row_ptr() const { return row.defined() ? row.data_ptr<int32_t>() : nullptr; }
};

void paged_append(const at::Tensor& kp, const at::Tensor& vp, const c10::optional<at::Tensor>& ks,
                  const c10::optional<at::Tensor>& vs, const at::Tensor& k_in, const at::Tensor& v_in,
                  const at::Tensor& table_in, const at::Tensor& positions, const c10::optional<at::Tensor>& rows,
                  int64_t st) {
  const char* who = "paged_append";
  const Cache c = cache_of(kp, vp, ks, vs, who);
  at::DeviceGuard guard(kp.device());
  no_tangents({k_in, v_in, kp, vp, c.ks, c.vs}, who);
  TORCH_CHECK(!wants_grad({k_in, v_in, kp, vp, c.ks, c.vs}), who, " has no backward: call it without gradients");
  at::NoGradGuard no_grad;
  const NewTokens n(c, k_in, v_in, table_in, positions, rows, who);
  const int64_t strides[4] = {row_stride(n.k), head_stride(n.k), row_stride(n.v), head_stride(n.v)};
  check(naylis_mom_paged_append(kp.data_ptr(), vp.data_ptr(), c.k_scale(), c.v_scale(), c.dtype, n.k.data_ptr(),
                                n.v.data_ptr(), strides, n.table.data_ptr<int32_t>(), n.pos.data_ptr<int32_t>(),
                                n.row_ptr(), n.T, c.pages, c.Hkv, c.page, c.hd, n.table.size(0), n.table.size(1),
                                stream_of(st, kp)));
  for (const at::Tensor& t : {c.k, c.v, c.ks, c.vs}) written(t);
}

// Returns the rotated queries (undefined without q).
at::Tensor paged_append_rope(const at::Tensor& kp, const at::Tensor& vp, const c10::optional<at::Tensor>& ks,
                             const c10::optional<at::Tensor>& vs, const c10::optional<at::Tensor>& q_in,
                             const at::Tensor& k_in, const at::Tensor& v_in, const at::Tensor& inv_freq,
                             const at::Tensor& table_in, const at::Tensor& positions,
                             const c10::optional<at::Tensor>& rows, double scaling, int64_t st) {
  const char* who = "paged_append_rope";
  const Cache c = cache_of(kp, vp, ks, vs, who);
  at::DeviceGuard guard(kp.device());
  const at::Tensor q_given = q_in.value_or(at::Tensor());
  no_tangents({q_given, k_in, v_in, inv_freq, kp, vp, c.ks, c.vs}, who);
  TORCH_CHECK(!wants_grad({q_given, k_in, v_in, inv_freq, kp, vp, c.ks, c.vs}), who,
              " has no backward: call it without gradients");
  at::NoGradGuard no_grad;
  const NewTokens n(c, k_in, v_in, table_in, positions, rows, who);
  same_device(inv_freq, kp, who, "inv_freq");
  TORCH_CHECK(inv_freq.dim() == 1 && inv_freq.scalar_type() == at::kFloat, who, ": inv_freq must be fp32 (half,), got ",
              inv_freq.sizes(), " ", inv_freq.scalar_type());
  const at::Tensor freq = inv_freq.contiguous();
  at::Tensor q, q_out;
  int64_t H = 0, strides[6] = {0, 0, row_stride(n.k), head_stride(n.k), row_stride(n.v), head_stride(n.v)};
  if (q_given.defined()) {
    same_device(q_given, kp, who, "q");
    TORCH_CHECK(q_given.dim() == 3 && q_given.scalar_type() == at::kBFloat16 && q_given.size(0) == n.T &&
                    q_given.size(1) > 0 && q_given.size(2) == c.hd,
                who, ": q must be bf16 (T, H, head_dim) of the same tokens; got ", q_given.sizes(), " ",
                q_given.scalar_type());
    q = rows_of(q_given);
    H = q.size(1);
    q_out = at::empty({n.T, H, c.hd}, q.options());
    strides[0] = row_stride(q);
    strides[1] = head_stride(q);
  }
  check(naylis_mom_paged_append_rope(kp.data_ptr(), vp.data_ptr(), c.k_scale(), c.v_scale(), c.dtype, ptr(q),
                                     n.k.data_ptr(), n.v.data_ptr(), strides, freq.data_ptr<float>(), (float)scaling,
                                     n.table.data_ptr<int32_t>(), n.pos.data_ptr<int32_t>(), n.row_ptr(), ptr(q_out),
                                     n.T, H, freq.size(0), c.pages, c.Hkv, c.page, c.hd, n.table.size(0),
                                     n.table.size(1), stream_of(st, kp)));
  for (const at::Tensor& t : {c.k, c.v, c.ks, c.vs}) written(t);
  return q_out;
}

variable_list paged_gather(const at::Tensor& kp, const at::Tensor& vp, const c10::optional<at::Tensor>& ks,
                           const c10::optional<at::Tensor>& vs, const at::Tensor& table_in, const at::Tensor& cu_in,
                           int64_t tokens, int64_t st) {
  const char* who = "paged_gather";
  const Cache c = cache_of(kp, vp, ks, vs, who);
  at::DeviceGuard guard(kp.device());
  no_tangents({kp, vp, c.ks, c.vs}, who);
  TORCH_CHECK(!wants_grad({kp, vp, c.ks, c.vs}), who, " has no backward: call it without gradients");
  at::NoGradGuard no_grad;
  const at::Tensor table = indices(table_in, kp, who, "block_table"), cu = indices(cu_in, kp, who, "cu_seqlens");
  TORCH_CHECK(table.dim() == 2 && table.size(0) > 0 && table.size(1) > 0 && cu.dim() == 1 &&
                  cu.size(0) == table.size(0) + 1,
              who, ": block_table must be (B, pages of a sequence) and cu_seqlens (B + 1,); got ", table.sizes(),
              " and ", cu.sizes());
  TORCH_CHECK(tokens >= 0, who, ": tokens must not be negative, got ", tokens);
  const at::TensorOptions o = kp.options().dtype(at::kBFloat16);
  at::Tensor k = at::empty({tokens, c.Hkv, c.hd}, o), v = at::empty({tokens, c.Hkv, c.hd}, o);
  check(naylis_mom_paged_gather(kp.data_ptr(), vp.data_ptr(), c.k_scale(), c.v_scale(), c.dtype,
                                table.data_ptr<int32_t>(), cu.data_ptr<int32_t>(), k.data_ptr(), v.data_ptr(), tokens,
                                c.pages, c.Hkv, c.page, c.hd, table.size(0), table.size(1), stream_of(st, kp)));
  return {k, v};
}

// A (B, N, H, hd) operand as the kernels read it; a dimension of one is not stepped over.
at::Tensor tokens_of(const at::Tensor& t, int64_t (&strides)[3]) {
  const auto fits = [&](const at::Tensor& x) {
    bool ok = x.stride(3) == 1 && (uintptr_t)x.data_ptr() % 16 == 0;
    for (int d = 0; d < 3; ++d) {
      strides[d] = x.size(d) > 1 ? x.stride(d) : 0;
      ok = ok && strides[d] % 8 == 0 && (d != 1 || strides[d] < (1 << 23));
    }
    return ok;
  };
  if (fits(t)) return t;
  at::Tensor c = t.contiguous();
  if ((uintptr_t)c.data_ptr() % 16 != 0) c = c.clone();
  fits(c);
  return c;
}

at::Tensor paged_attention(const at::Tensor& q_in, const at::Tensor& kp, const at::Tensor& vp,
                           const c10::optional<at::Tensor>& ks, const c10::optional<at::Tensor>& vs,
                           const at::Tensor& table_in, const at::Tensor& lens_in, c10::optional<double> scale,
                           const c10::optional<at::Tensor>& q_lens, int64_t st) {
  const char* who = "paged_attention";
  const Cache c = cache_of(kp, vp, ks, vs, who);
  at::DeviceGuard guard(kp.device());
  no_tangents({q_in, kp, vp, c.ks, c.vs}, who);
  TORCH_CHECK(!wants_grad({q_in, kp, vp, c.ks, c.vs}), who, " has no backward: call it without gradients");
  at::NoGradGuard no_grad;
  const bool many = q_in.dim() == 4;
  const int64_t heads = many ? 2 : 1;
  TORCH_CHECK((many || q_in.dim() == 3) && q_in.scalar_type() == at::kBFloat16 && q_in.size(heads + 1) == c.hd &&
                  c.Hkv > 0 && q_in.size(heads) > 0 && q_in.size(heads) % c.Hkv == 0 && q_in.size(heads - 1) >= (many ? 1 : 0),
              who, ": q must be bf16 (B, H, head_dim) or (B, N, H, head_dim) with N >= 1 and H a multiple of the ",
              "cache's heads; got ", q_in.sizes(), " ", q_in.scalar_type(), " for a cache of ", c.k.sizes());
  same_device(q_in, kp, who, "q");
  const at::Tensor table = indices(table_in, kp, who, "block_table"), lens = indices(lens_in, kp, who, "seq_lens");
  const int64_t B = q_in.size(0), N = many ? q_in.size(1) : 1, H = q_in.size(heads);
  TORCH_CHECK(table.dim() == 2 && table.size(0) == B && table.size(1) > 0 && lens.dim() == 1 && lens.size(0) == B,
              who, ": block_table must be (B, pages of a sequence) and seq_lens (B,) for the ", B, " rows of q");
  at::Tensor live;
  if (q_lens.has_value()) {
    live = indices(*q_lens, kp, who, "q_lens");
    TORCH_CHECK(live.dim() == 1 && live.size(0) == B, who, ": q_lens must be (B,) for the ", B, " rows of q");
  }
  int64_t strides[3];
  const at::Tensor q = tokens_of(many ? q_in : q_in.unsqueeze(1), strides);
  at::Tensor out = at::empty(q_in.sizes(), q_in.options().memory_format(at::MemoryFormat::Contiguous));
  const size_t bytes = naylis_mom_paged_attn_tokens_workspace_bytes(c.dtype, B, N, H, c.Hkv, c.page, c.hd, table.size(1));
  const at::Tensor ws = bytes ? workspace(bytes, q) : at::Tensor();
  check(naylis_mom_paged_attn_tokens(q.data_ptr(), kp.data_ptr(), vp.data_ptr(), c.k_scale(), c.v_scale(), c.dtype,
                                     table.data_ptr<int32_t>(), lens.data_ptr<int32_t>(),
                                     live.defined() ? live.data_ptr<int32_t>() : nullptr, out.data_ptr(), ptr(ws),
                                     bytes, strides, (float)scale_of(scale, c.hd), B, N, H, c.pages, c.Hkv, c.page,
                                     c.hd, table.size(1), stream_of(st, kp)));
  return out;
}

// ---- log probabilities ------------------------------------------------------------

// (N, V) rows of dense elements
at::Tensor logit_rows(const at::Tensor& logits) {
  const at::Tensor x = logits.reshape({-1, logits.size(-1)});
  return x.size(1) == 1 || x.stride(1) == 1 ? x : x.contiguous();
}

variable_list logprobs_forward(const at::Tensor& x, const at::Tensor& tokens, int64_t top, int64_t ignore_index,
                               at::Tensor* stat, void* st) {
  const int64_t N = x.size(0), V = x.size(1);
  at::Tensor logp = at::empty({N}, f32_like(x)), entropy = at::empty({N}, f32_like(x));
  at::Tensor ids = at::empty({N, top}, x.options().dtype(at::kLong)), lps = at::empty({N, top}, f32_like(x));
  if (stat) *stat = at::empty({N, 3}, f32_like(x));
  const size_t bytes = naylis_mom_logprobs_workspace_bytes(N, V, top);
  const at::Tensor ws = bytes ? workspace(bytes, x) : at::Tensor();
  check(naylis_mom_logprobs_fwd(x.data_ptr(), dtype_code(x), x.stride(0), tokens.data_ptr<int64_t>(),
                                logp.data_ptr<float>(), entropy.data_ptr<float>(),
                                stat ? stat->data_ptr<float>() : nullptr, ids.data_ptr<int64_t>(),
                                lps.data_ptr<float>(), ptr(ws), bytes, N, V, top, ignore_index, st));
  return {logp, entropy, ids, lps};
}

// fp32 gradient of one value a row, as it is where it is one value for all rows
struct RowGrad {
  at::Tensor t;
  int64_t stride = 0;
  explicit RowGrad(const at::Tensor& g) {
    if (!g.defined()) return;
    t = g.to(at::kFloat);
    if (t.dim() != 1 || t.stride(0) != 0) t = t.contiguous();
    stride = t.stride(0);
  }
  const float* ptr() const { return t.defined() ? t.data_ptr<float>() : nullptr; }
};

at::Tensor logprobs_grad(const at::Tensor& x, const at::Tensor& tokens, const at::Tensor& stat, const at::Tensor& gl,
                         const at::Tensor& ge, int64_t ignore_index) {
  at::DeviceGuard guard(x.device());
  const RowGrad a(gl), b(ge);
  at::Tensor dx = at::empty({x.size(0), x.size(1)}, x.options());
  check(naylis_mom_logprobs_bwd(x.data_ptr(), dtype_code(x), x.stride(0), tokens.data_ptr<int64_t>(),
                                stat.data_ptr<float>(), a.ptr(), a.stride, b.ptr(), b.stride, dx.data_ptr(),
                                x.size(0), x.size(1), ignore_index, current_stream(x)));
  return dx;
}

struct LogprobsGrad : public Function<LogprobsGrad> {
  static at::Tensor forward(AutogradContext*, at::Tensor x, at::Tensor tokens, at::Tensor stat, at::Tensor gl,
                            at::Tensor ge, int64_t ignore_index) {
    return logprobs_grad(x, tokens, stat, gl, ge, ignore_index);
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "token_logprobs: the derivative of its backward is not implemented");
  }
};

struct Logprobs : public Function<Logprobs> {
  static variable_list forward(AutogradContext* ctx, at::Tensor x, at::Tensor tokens, int64_t top,
                               int64_t ignore_index, int64_t st) {
    at::Tensor stat;
    variable_list out = logprobs_forward(x, tokens, top, ignore_index, &stat, stream_ptr(st));
    ctx->save_for_backward({x, tokens, stat});
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->mark_non_differentiable({out[2], out[3]});
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const int64_t ignore_index = ctx->saved_data["ignore_index"].toInt();
    at::Tensor dx;
    if (at::GradMode::is_enabled()) {
      auto given = [&](const at::Tensor& g) { return g.defined() ? g : at::zeros({s[0].size(0)}, f32_like(s[0])); };
      dx = LogprobsGrad::apply(s[0], s[1], s[2], given(grads[0]), given(grads[1]), ignore_index);
    } else {
      dx = logprobs_grad(s[0], s[1], s[2], grads[0], grads[1], ignore_index);
    }
    return {dx, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

variable_list token_logprobs(const at::Tensor& logits, const at::Tensor& tokens_in, int64_t top, int64_t ignore_index,
                             int64_t stream) {
  const char* who = "token_logprobs";
  on_gpu(logits, who, "logits");
  at::DeviceGuard guard(logits.device());
  TORCH_CHECK(logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kFloat, who,
              ": logits must be bf16 or fp32, got ", logits.scalar_type());
  TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) > 0 && tokens_in.sizes() == logits.sizes().slice(0, logits.dim() - 1),
              who, ": needs logits (..., V) and tokens (...); got ", logits.sizes(), " and ", tokens_in.sizes());
  TORCH_CHECK(top >= 0 && top <= logits.size(-1), who, ": top ", top, " must be in [0, V]");
  same_device(tokens_in, logits, who, "tokens");
  TORCH_CHECK(tokens_in.scalar_type() == at::kLong || tokens_in.scalar_type() == at::kInt, who,
              ": tokens must be int64 or int32");
  no_tangents({logits}, who);
  const at::Tensor tokens = tokens_in.reshape({-1}).to(at::kLong).contiguous();
  const at::Tensor x = logit_rows(logits);  // part of the graph where it copies
  void* st = stream_of(stream, logits);
  variable_list out;
  if (wants_grad({logits})) {
    out = Logprobs::apply(x, tokens, top, ignore_index, reinterpret_cast<int64_t>(st));
  } else {
    at::NoGradGuard no_grad;
    out = logprobs_forward(x, tokens, top, ignore_index, nullptr, st);
  }
  if (logits.dim() == 2) return out;
  std::vector<int64_t> lead = tokens_in.sizes().vec(), tops = lead;
  tops.push_back(top);
  return {out[0].view(lead), out[1].view(lead), out[2].view(tops), out[3].view(tops)};
}

// ---- drafts' verification ---------------------------------------------------------

// (B, n, V) of dense rows
at::Tensor dense_rows(const at::Tensor& t, int64_t (&strides)[2]) {
  const at::Tensor x = t.size(2) == 1 || t.stride(2) == 1 ? t : t.contiguous();
  strides[0] = x.size(0) == 1 ? 0 : x.stride(0);
  strides[1] = x.size(1) == 1 ? 0 : x.stride(1);
  return x;
}

variable_list verify_drafts(const at::Tensor& logits_in, const at::Tensor& drafts_in, const at::Tensor& uniforms_in,
                            const c10::optional<at::Tensor>& probs_in, const c10::optional<at::Tensor>& lens_in,
                            const c10::optional<at::Tensor>& temps_in, double temperature, int64_t st) {
  const char* who = "verify_drafts";
  on_gpu(logits_in, who, "logits");
  at::DeviceGuard guard(logits_in.device());
  const auto real = [](const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; };
  TORCH_CHECK(logits_in.dim() == 3 && real(logits_in) && logits_in.size(1) > 0 && logits_in.size(2) > 0, who,
              ": logits must be bf16 or fp32 (B, N + 1, V), got ", logits_in.sizes(), " ", logits_in.scalar_type());
  const int64_t B = logits_in.size(0), N = logits_in.size(1) - 1, V = logits_in.size(2);
  same_device(drafts_in, logits_in, who, "drafts");
  same_device(uniforms_in, logits_in, who, "uniforms");
  TORCH_CHECK(drafts_in.dim() == 2 && drafts_in.size(0) == B && drafts_in.size(1) == N &&
                  (drafts_in.scalar_type() == at::kLong || drafts_in.scalar_type() == at::kInt),
              who, ": drafts must be int64 or int32 (B, N) for logits (B, N + 1, V); got ", drafts_in.sizes(), " ",
              drafts_in.scalar_type(), " for ", logits_in.sizes());
  TORCH_CHECK(uniforms_in.dim() == 2 && uniforms_in.size(0) == B && uniforms_in.size(1) == N + 1 &&
                  uniforms_in.scalar_type() == at::kFloat,
              who, ": uniforms must be fp32 (B, N + 1); got ", uniforms_in.sizes(), " ", uniforms_in.scalar_type());
  const at::Tensor probs_given = probs_in.value_or(at::Tensor()), temps_given = temps_in.value_or(at::Tensor());
  no_tangents({logits_in, uniforms_in, probs_given, temps_given}, who);
  TORCH_CHECK(!wants_grad({logits_in, uniforms_in, probs_given, temps_given}), who,
              " has no backward: call it without gradients");
  at::NoGradGuard no_grad;
  int64_t strides[2], probs_strides[2] = {0, 0};
  const at::Tensor logits = dense_rows(logits_in, strides), drafts = drafts_in.to(at::kLong).contiguous();
  const at::Tensor uniforms = uniforms_in.contiguous();
  at::Tensor probs, lens, temps;
  if (probs_given.defined()) {
    same_device(probs_given, logits, who, "draft_probs");
    TORCH_CHECK(probs_given.dim() == 3 && real(probs_given) && probs_given.size(0) == B && probs_given.size(1) == N &&
                    probs_given.size(2) == V,
                who, ": draft_probs must be bf16 or fp32 (B, N, V); got ", probs_given.sizes(), " ",
                probs_given.scalar_type());
    if (N > 0) probs = dense_rows(probs_given, probs_strides);
  }
  if (lens_in.has_value()) {
    lens = indices(*lens_in, logits, who, "draft_lens");
    TORCH_CHECK(lens.dim() == 1 && lens.size(0) == B, who, ": draft_lens must be (B,)");
  }
  if (temps_given.defined()) {
    same_device(temps_given, logits, who, "temperature");
    TORCH_CHECK(temps_given.dim() == 1 && temps_given.size(0) == B && temps_given.scalar_type() == at::kFloat, who,
                ": temperature must be a number or fp32 (B,)");
    temps = temps_given.contiguous();
  }
  at::Tensor tokens = at::empty({B, N + 1}, logits.options().dtype(at::kLong));
  at::Tensor accepted = at::empty({B}, logits.options().dtype(at::kInt));
  const size_t bytes = naylis_mom_verify_drafts_workspace_bytes(B, N, V, probs.defined());
  const at::Tensor ws = bytes ? workspace(bytes, logits) : at::Tensor();
  check(naylis_mom_verify_drafts(logits.data_ptr(), dtype_code(logits), strides, drafts.data_ptr<int64_t>(),
                                 uniforms.data_ptr<float>(), ptr(probs), probs.defined() ? dtype_code(probs) : kF32,
                                 probs_strides, lens.defined() ? lens.data_ptr<int32_t>() : nullptr,
                                 temps.defined() ? temps.data_ptr<float>() : nullptr, (float)temperature,
                                 tokens.data_ptr<int64_t>(), accepted.data_ptr<int32_t>(), ptr(ws), bytes, B, N,
                                 V, stream_of(st, logits)));
  return {tokens, accepted};
}

}  // namespace

void bind_serving(pybind11::module_& m) {
  m.def("packed_attention", &packed_attention);
  m.def("paged_append", &paged_append);
  m.def("paged_attention", &paged_attention);
  m.def("paged_append_rope", &paged_append_rope);
  m.def("paged_gather", &paged_gather);
  m.def("token_logprobs", &token_logprobs);
  m.def("verify_drafts", &verify_drafts);
}

}  // namespace naylis_ext
