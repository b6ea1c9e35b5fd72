// Packed attention, the paged cache and token log probabilities: argument
// checks, the C-ABI calls and the autograd nodes behind
// mom_kernels/hip_packed.py, hip_paged.py and hip_logprobs.py.  Calls without
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

constexpr int kE4M3 = 2;

struct Cache {
  at::Tensor k, v, ks, vs;
  int dtype;
  int64_t pages, Hkv, page, hd;
  float* k_scale() const { return ks.defined() ? ks.data_ptr<float>() : nullptr; }
  float* v_scale() const { return vs.defined() ? vs.data_ptr<float>() : nullptr; }
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
              ": the cache must be bf16, or e4m3 codes in uint8 with scales; got ", k.scalar_type());
  TORCH_CHECK(codes == ks.has_value() && codes == vs.has_value(), who,
              ": e4m3 pages need k_scale and v_scale, bf16 pages have none");
  Cache c{k, v, ks.value_or(at::Tensor()), vs.value_or(at::Tensor()), codes ? kE4M3 : kBF16,
          k.size(0), k.size(1), k.size(2), k.size(3)};
  if (codes)
    for (const at::Tensor& s : {c.ks, c.vs})
      TORCH_CHECK(s.scalar_type() == at::kFloat && s.is_contiguous() && s.device() == k.device() &&
                      s.sizes() == k.sizes().slice(0, 3) && (uintptr_t)s.data_ptr() % 16 == 0,
                  who, ": k_scale and v_scale must be dense fp32 (pages, Hkv, page_size) tensors, 16-byte aligned");
  return c;
}

void written(const at::Tensor& t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

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
  TORCH_CHECK(k_in.dim() == 3 && v_in.sizes() == k_in.sizes() && k_in.size(1) == c.Hkv && k_in.size(2) == c.hd &&
                  k_in.scalar_type() == at::kBFloat16 && v_in.scalar_type() == at::kBFloat16,
              who, ": k and v must be bf16 (T, Hkv, head_dim) of the cache's heads; got ", k_in.sizes(), " ",
              k_in.scalar_type(), ", ", v_in.sizes(), " ", v_in.scalar_type());
  same_device(k_in, kp, who, "k");
  same_device(v_in, kp, who, "v");
  const at::Tensor table = indices(table_in, kp, who, "block_table"), pos = indices(positions, kp, who, "positions");
  const at::Tensor row = rows.has_value() ? indices(*rows, kp, who, "rows") : at::Tensor();
  const int64_t T = k_in.size(0);
  TORCH_CHECK(table.dim() == 2 && table.size(1) > 0, who, ": block_table must be (B, pages of a sequence)");
  TORCH_CHECK(pos.dim() == 1 && pos.size(0) == T && (!row.defined() || row.sizes() == pos.sizes()), who,
              ": positions and rows must hold one entry for each of the ", T, " tokens");
  const at::Tensor k = rows_of(k_in), v = rows_of(v_in);
  const int64_t strides[4] = {row_stride(k), head_stride(k), row_stride(v), head_stride(v)};
  check(naylis_mom_paged_append(kp.data_ptr(), vp.data_ptr(), c.k_scale(), c.v_scale(), c.dtype, k.data_ptr(),
                                v.data_ptr(), strides, table.data_ptr<int32_t>(), pos.data_ptr<int32_t>(),
                                row.defined() ? row.data_ptr<int32_t>() : nullptr, T, c.pages, c.Hkv, c.page, c.hd,
                                table.size(0), table.size(1), stream_of(st, kp)));
  for (const at::Tensor& t : {c.k, c.v, c.ks, c.vs}) written(t);
}

at::Tensor paged_attention(const at::Tensor& q_in, const at::Tensor& kp, const at::Tensor& vp,
                           const c10::optional<at::Tensor>& ks, const c10::optional<at::Tensor>& vs,
                           const at::Tensor& table_in, const at::Tensor& lens_in, c10::optional<double> scale,
                           int64_t st) {
  const char* who = "paged_attention";
  const Cache c = cache_of(kp, vp, ks, vs, who);
  at::DeviceGuard guard(kp.device());
  no_tangents({q_in, kp, vp, c.ks, c.vs}, who);
  TORCH_CHECK(!wants_grad({q_in, kp, vp, c.ks, c.vs}), who, " has no backward: call it without gradients");
  at::NoGradGuard no_grad;
  TORCH_CHECK(q_in.dim() == 3 && q_in.scalar_type() == at::kBFloat16 && q_in.size(2) == c.hd && c.Hkv > 0 &&
                  q_in.size(1) > 0 && q_in.size(1) % c.Hkv == 0,
              who, ": q must be bf16 (B, H, head_dim) with H a multiple of the cache's heads; got ", q_in.sizes(), " ",
              q_in.scalar_type(), " for a cache of ", c.k.sizes());
  same_device(q_in, kp, who, "q");
  const at::Tensor table = indices(table_in, kp, who, "block_table"), lens = indices(lens_in, kp, who, "seq_lens");
  const int64_t B = q_in.size(0), H = q_in.size(1);
  TORCH_CHECK(table.dim() == 2 && table.size(0) == B && table.size(1) > 0 && lens.dim() == 1 && lens.size(0) == B,
              who, ": block_table must be (B, pages of a sequence) and seq_lens (B,) for the ", B, " rows of q");
  const at::Tensor q = rows_of(q_in);
  at::Tensor out = at::empty({B, H, c.hd}, q.options());
  const size_t bytes = naylis_mom_paged_attn_workspace_bytes(c.dtype, B, H, c.Hkv, c.page, c.hd, table.size(1));
  const at::Tensor ws = bytes ? workspace(bytes, q) : at::Tensor();
  const int64_t strides[2] = {row_stride(q), head_stride(q)};
  check(naylis_mom_paged_attn(q.data_ptr(), kp.data_ptr(), vp.data_ptr(), c.k_scale(), c.v_scale(), c.dtype,
                              table.data_ptr<int32_t>(), lens.data_ptr<int32_t>(), out.data_ptr(), ptr(ws), bytes,
                              strides, (float)scale_of(scale, c.hd), B, H, c.pages, c.Hkv, c.page, c.hd,
                              table.size(1), stream_of(st, kp)));
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

}  // namespace

void bind_serving(pybind11::module_& m) {
  m.def("packed_attention", &packed_attention);
  m.def("paged_append", &paged_append);
  m.def("paged_attention", &paged_attention);
  m.def("token_logprobs", &token_logprobs);
}

}  // namespace naylis_ext
