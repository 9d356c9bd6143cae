// Torch binding of the latent attention (axiom_amd/latent.py): argument checks,
// outputs and workspaces, the call of include/latent_mi355x.h on torch's current
// stream, and the differentiable form as a C++ autograd function.
//
// A small call costs what its host path costs: the same checks in Python and a
// ctypes call took 11.7 us around a 5 us kernel (prompt of 512 tokens), and a
// Python backward another thread's turn with the interpreter.

#include "torch_binding.h"

void bind_tree(py::module_& m);   // tree_torch.cpp

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// sizes, strides and packed offsets of an expanded-form call
struct Attn {
  int B, Tq, Tk, H, dn, dr, n_seqs = 0, code;
  int64_t strides[8];
  OptTensor cu_q, cu_k;
  double scale;
};

Attn attn_check(const char* what, const Tensor& q, const Tensor& kv, const Tensor& kr, const OptTensor& cu_q, const OptTensor& cu_k,
                std::optional<double> scale) {
  if (q.dim() != 4 || kv.dim() != 4 || kr.dim() != 3)
    refuse(what, "q must be [B,Tq,H,dn+dr], kv [B,Tk,H,2 dn], k_rope [B,Tk,dr]");
  const int64_t B = q.size(0), Tq = q.size(1), H = q.size(2), Tk = kv.size(1), dn = kv.size(3) / 2, dr = kr.size(2);
  if (kv.size(0) != B || kv.size(2) != H || kv.size(3) != 2 * dn || kr.size(0) != B || kr.size(1) != Tk || q.size(3) != dn + dr)
    refuse(what, "q ", q.sizes(), ", kv ", kv.sizes(), " and k_rope ", kr.sizes(),
           " do not fit q [B,Tq,H,dn+dr], kv [B,Tk,H,2 dn], k_rope [B,Tk,dr]");
  if (std::max({B, Tq, Tk, H, dn}) > INT32_MAX) refuse(what, "sizes past 2^31");
  Attn a;
  a.B = B; a.Tq = Tq; a.Tk = Tk; a.H = H; a.dn = dn; a.dr = dr;
  a.code = code_of(q);
  if (a.code < 0 || kv.scalar_type() != q.scalar_type() || kr.scalar_type() != q.scalar_type())
    refuse(what, "q, kv, k_rope must share a dtype in bf16/fp16/fp32");
  if ((dn + dr > 1 && q.stride(3) != 1) || (dn > 0 && kv.stride(3) != 1) || (dr > 1 && kr.stride(2) != 1))
    refuse(what, "the last axis of q, kv and k_rope must be contiguous");
  const int64_t st[8] = {q.stride(0), q.stride(1), q.stride(2), kv.stride(0), kv.stride(1), kv.stride(2), kr.stride(0), kr.stride(1)};
  std::copy(st, st + 8, a.strides);
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  if (cu_q) {
    if (!cu_k) {
      if (Tq != Tk) refuse(what, "cu_seqlens alone needs Tq == Tk, got ", Tq, " and ", Tk);
      a.cu_k = cu_q;
    }
    for (const OptTensor* cu : {&a.cu_q, &a.cu_k}) {
      const char* name = cu == &a.cu_q ? "cu_seqlens" : "cu_seqlens_k";
      if ((*cu)->scalar_type() != at::kInt || (*cu)->dim() != 1 || (*cu)->numel() < 2)
        refuse(what, name, " must be a 1-D int32 tensor of N+1 >= 2 offsets");
      contiguous(name, **cu);
    }
    if (a.cu_q->numel() != a.cu_k->numel()) refuse(what, "cu_seqlens and cu_seqlens_k must have the same length");
    if (B != 1) refuse(what, "cu_seqlens requires B == 1, got B=", B);
    a.n_seqs = static_cast<int>(a.cu_q->numel() - 1);
  } else if (cu_k) {
    refuse(what, "cu_seqlens_k requires cu_seqlens");
  }
  a.scale = scale ? *scale : 1.0 / std::sqrt(static_cast<double>(dn + dr));
  return a;
}

std::tuple<Tensor, Tensor> attn_fwd(const Tensor& q, const Tensor& kv, const Tensor& kr, const OptTensor& cu_q, const OptTensor& cu_k,
                                    bool causal, std::optional<double> scale, const OptTensor& out, const OptTensor& lse_out,
                                    const OptTensor& workspace) {
  const char* what = "latent_attn_fwd";
  const Attn a = attn_check(what, q, kv, kr, cu_q, cu_k, scale);
  const at::Device d = one_gpu(what, q, kv, kr, a.cu_q, a.cu_k);
  const c10::DeviceGuard on(d);
  Tensor o = output(what, "out", out, {a.B, a.Tq, a.H, a.dn}, q.scalar_type(), d);
  Tensor lse = output(what, "lse", lse_out, {a.B, a.H, a.Tq}, at::kFloat, d);
  const size_t bytes = kda_latent_attn_fwd_workspace(a.B, a.Tq, a.Tk, a.H, a.dn, a.dr, a.n_seqs, a.code);
  const Tensor ws = work(workspace, bytes, d);
  checked(kda_latent_attn_fwd(stream_of(d), ptr(q), ptr(kv), ptr(kr), a.strides, static_cast<const int32_t*>(ptr(a.cu_q)),
                              static_cast<const int32_t*>(ptr(a.cu_k)), a.n_seqs, ptr(o), static_cast<float*>(ptr(lse)), a.B, a.Tq,
                              a.Tk, a.H, a.dn, a.dr, causal, static_cast<float>(a.scale), a.code, work_ptr(ws), bytes),
          what);
  written(out);
  written(lse_out);
  return {o, lse};
}

std::tuple<Tensor, Tensor, Tensor> attn_bwd(const Tensor& q, const Tensor& kv, const Tensor& kr, const Tensor& o, const Tensor& lse,
                                            const Tensor& d_o, const OptTensor& cu_q, const OptTensor& cu_k, bool causal,
                                            std::optional<double> scale, const OptTensor& workspace) {
  const char* what = "latent_attn_bwd";
  const Attn a = attn_check(what, q, kv, kr, cu_q, cu_k, scale);
  const int64_t shape[4] = {a.B, a.Tq, a.H, a.dn}, rows[3] = {a.B, a.H, a.Tq};
  for (const Tensor* t : {&o, &d_o}) {
    const char* name = t == &o ? "o" : "do";
    if (t->sizes() != at::IntArrayRef(shape, 4) || t->scalar_type() != q.scalar_type())
      refuse(what, name, " must be ", q.scalar_type(), " ", at::IntArrayRef(shape, 4));
    contiguous(name, *t);
  }
  if (lse.sizes() != at::IntArrayRef(rows, 3) || lse.scalar_type() != at::kFloat) refuse(what, "lse must be fp32 ", at::IntArrayRef(rows, 3));
  contiguous("lse", lse);
  const at::Device d = one_gpu(what, q, kv, kr, o, lse, d_o, a.cu_q, a.cu_k);
  const c10::DeviceGuard on(d);
  const size_t bytes = kda_latent_attn_bwd_workspace(a.B, a.Tq, a.Tk, a.H, a.dn, a.dr, a.n_seqs, a.code);
  const Tensor ws = work(workspace, bytes, d);
  const auto opt = q.options().requires_grad(false);
  Tensor dq = at::empty({a.B, a.Tq, a.H, a.dn + a.dr}, opt), dkv = at::empty({a.B, a.Tk, a.H, 2 * a.dn}, opt);
  Tensor dkr = at::empty({a.B, a.Tk, a.dr}, opt);
  checked(kda_latent_attn_bwd(stream_of(d), ptr(q), ptr(kv), ptr(kr), a.strides, static_cast<const int32_t*>(ptr(a.cu_q)),
                              static_cast<const int32_t*>(ptr(a.cu_k)), a.n_seqs, ptr(o), static_cast<const float*>(ptr(lse)), ptr(d_o),
                              ptr(dq), ptr(dkv), ptr(dkr), a.B, a.Tq, a.Tk, a.H, a.dn, a.dr, causal, static_cast<float>(a.scale),
                              a.code, work_ptr(ws), bytes),
          what);
  return {dq, dkv, dkr};
}

struct LatentAttn : torch::autograd::Function<LatentAttn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& kv, const Tensor& kr, const OptTensor& cu_q,
                        const OptTensor& cu_k, bool causal, double scale) {
    const auto [o, lse] = attn_fwd(q, kv, kr, cu_q, cu_k, causal, scale, std::nullopt, std::nullopt, std::nullopt);
    variable_list kept = {q, kv, kr, o, lse};
    if (cu_q) kept.push_back(*cu_q);
    if (cu_k) kept.push_back(*cu_k);
    ctx->save_for_backward(std::move(kept));
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(7);
    if (!grads[0].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    const OptTensor cu_q = s.size() > 5 ? OptTensor(s[5]) : std::nullopt, cu_k = s.size() > 6 ? OptTensor(s[6]) : std::nullopt;
    std::tie(out[0], out[1], out[2]) = attn_bwd(s[0], s[1], s[2], s[3], s[4], grads[0].contiguous(), cu_q, cu_k,
                                                ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble(), std::nullopt);
    // create_graph: the gradients are the kernels' and have no derivative of their
    // own; differentiating them by what they were made from raises instead of
    // leaving terms out
    if (at::GradMode::is_enabled()) {
      const auto once = std::make_shared<torch::autograd::Error>("latent_attn is not differentiable twice",
                                                                 torch::autograd::collect_next_edges(s[0], s[1], s[2], grads[0]));
      for (int i = 0; i < 3; ++i) torch::autograd::create_gradient_edge(out[i], once);
    }
    return out;
  }
};

Tensor attn(const Tensor& q, const Tensor& kv, const Tensor& kr, const OptTensor& cu_q, const OptTensor& cu_k, bool causal,
            std::optional<double> scale) {
  const Attn a = attn_check("latent_attn", q, kv, kr, cu_q, cu_k, scale);
  return LatentAttn::apply(q, kv, kr, cu_q, cu_k, causal, a.scale);
}

OptTensor append(const Tensor& rows, const Tensor& positions, const Tensor& slots, const Tensor& cos_sin, Tensor cache,
                 const OptTensor& weight, double eps, const OptTensor& q, OptTensor q_out, bool interleaved) {
  const char* what = "latent_append";
  if (rows.dim() != 2 || cache.dim() != 3 || cache.size(2) != rows.size(1))
    refuse(what, "rows must be [N, R+dr] and cache [n_pages, page_size, R+dr]");
  if (cos_sin.dim() != 2 || cos_sin.scalar_type() != at::kFloat || cos_sin.size(0) < 1) refuse(what, "cos_sin must be fp32 [P, dr]");
  const int64_t N = rows.size(0), dr = cos_sin.size(1), R = rows.size(1) - dr;
  const int code = code_of(rows);
  if (code < 0 || cache.scalar_type() != rows.scalar_type()) refuse(what, "rows and cache must share a dtype in bf16/fp16/fp32");
  if (N > INT32_MAX || R > INT32_MAX || dr > INT32_MAX) refuse(what, "sizes past 2^31");
  for (const Tensor* t : {&positions, &slots}) {
    const char* name = t == &positions ? "positions" : "slots";
    if (t->scalar_type() != at::kLong || t->dim() != 1 || t->size(0) != N) refuse(what, name, " must be int64 [", N, "]");
    contiguous(name, *t);
  }
  if (weight) {
    if (weight->scalar_type() != at::kFloat || weight->dim() != 1 || weight->size(0) != R) refuse(what, "norm_weight must be fp32 [", R, "]");
    contiguous("norm_weight", *weight);
  }
  contiguous("cos_sin", cos_sin);
  contiguous("cache", cache);
  if (rows.stride(1) != 1) refuse(what, "the last axis of rows must be contiguous");
  int64_t H = 0, st[4] = {0, 0, 0, 0};
  if (q) {
    if (q->dim() != 3 || q->size(0) != N || q->size(2) != dr || q->scalar_type() != rows.scalar_type())
      refuse(what, "q_rope must be ", rows.scalar_type(), " [", N, ", H, ", dr, "]");
    H = q->size(1);
    if (H == 0 || H > INT32_MAX) refuse(what, "q_rope has no heads");
    if (!q_out) q_out = at::empty(q->sizes(), q->options().requires_grad(false));
    if (q_out->sizes() != q->sizes() || q_out->scalar_type() != q->scalar_type()) refuse(what, "q_out must match q_rope");
    if (q->stride(2) != 1 || q_out->stride(2) != 1) refuse(what, "the last axis of q_rope and q_out must be contiguous");
    st[0] = q->stride(0); st[1] = q->stride(1); st[2] = q_out->stride(0); st[3] = q_out->stride(1);
  } else if (q_out) {
    refuse(what, "q_out requires q_rope");
  }
  const at::Device d = one_gpu(what, rows, positions, slots, cos_sin, cache, weight, q, q_out);
  const c10::DeviceGuard on(d);
  checked(kda_latent_append(stream_of(d), ptr(rows), rows.stride(0), static_cast<const int64_t*>(ptr(positions)),
                            static_cast<const int64_t*>(ptr(slots)), static_cast<const float*>(ptr(cos_sin)), cos_sin.size(0),
                            static_cast<const float*>(ptr(weight)), static_cast<float>(eps), ptr(cache), cache.size(0) * cache.size(1),
                            ptr(q), st[0], st[1], ptr(q_out), st[2], st[3], static_cast<int>(N), static_cast<int>(H),
                            static_cast<int>(R), static_cast<int>(dr), interleaved, code),
          what);
  written(cache);
  written(q_out);
  return q_out;
}

std::tuple<Tensor, Tensor> decode(const Tensor& q, const Tensor& cache, const Tensor& table, const Tensor& lens, double scale,
                                  const OptTensor& out, const OptTensor& lse_out, const OptTensor& workspace) {
  const char* what = "latent_decode";
  if (q.dim() != 4 || cache.dim() != 3 || q.size(3) != cache.size(2))
    refuse(what, "q must be [B,Tq,H,R+dr] and cache [n_pages, page_size, R+dr]");
  const int64_t B = q.size(0), Tq = q.size(1), H = q.size(2), W = q.size(3), R = W > 512 ? 512 : 256;
  const int code = code_of(q);
  if (code < 0 || cache.scalar_type() != q.scalar_type()) refuse(what, "q and cache must share a dtype in bf16/fp16/fp32");
  if (table.dim() != 2 || table.size(0) != B || table.scalar_type() != at::kInt) refuse(what, "block_table must be int32 [", B, ", max_pages]");
  if (lens.dim() != 1 || lens.size(0) != B || lens.scalar_type() != at::kInt) refuse(what, "seq_lens must be int32 [", B, "]");
  if (std::max({B, Tq, H, W, cache.size(1), table.size(1)}) > INT32_MAX) refuse(what, "sizes past 2^31");
  contiguous("q", q);
  contiguous("cache", cache);
  contiguous("block_table", table);
  contiguous("seq_lens", lens);
  const at::Device d = one_gpu(what, q, cache, table, lens);
  const c10::DeviceGuard on(d);
  const int page = static_cast<int>(cache.size(1)), per = static_cast<int>(table.size(1));
  const size_t bytes = kda_latent_decode_workspace(B, Tq, H, R, W - R, page, per, code);
  const Tensor ws = work(workspace, bytes, d);
  Tensor o = output(what, "out", out, {B, Tq, H, R}, q.scalar_type(), d);
  Tensor lse = output(what, "lse", lse_out, {B, Tq, H}, at::kFloat, d);
  checked(kda_latent_decode(stream_of(d), ptr(q), ptr(cache), static_cast<const int32_t*>(ptr(table)), static_cast<const int32_t*>(ptr(lens)),
                            ptr(o), static_cast<float*>(ptr(lse)), B, Tq, H, R, W - R, cache.size(0), page, per,
                            static_cast<float>(scale), code, work_ptr(ws), bytes),
          what);
  written(out);
  written(lse_out);
  return {o, lse};
}

}  // namespace

PYBIND11_MODULE(_latent_torch, m) {
  m.def("attn_fwd", &attn_fwd);
  m.def("attn_bwd", &attn_bwd);
  m.def("attn", &attn);
  m.def("append", &append);
  m.def("decode", &decode);
  bind_tree(m);
}
