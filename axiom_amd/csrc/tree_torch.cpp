// Torch binding of the tree calls (axiom_amd/tree.py): argument checks, outputs and
// workspaces, the call of include/tree_mi355x.h on torch's current stream.  In C++
// as the latent attention's, and in the same module: the checks are part of what
// a call of a few microseconds costs.

#include "torch_binding.h"

namespace {

const int32_t* i32(const Tensor& t) { return static_cast<const int32_t*>(ptr(t)); }

void places(const char* what, const Tensor& parents, int64_t B, int64_t N) {
  if (parents.dim() != 2 || parents.size(0) != B || parents.size(1) != N || parents.scalar_type() != at::kInt)
    refuse(what, "parents must be int32 [", B, ", ", N, "]");
  if (N < 1 || N > 64) refuse(what, "a tree has 1 to 64 places, got ", N);
  contiguous("parents", parents);
}
void per_sequence(const char* what, const char* name, const Tensor& t, int64_t B) {
  if (t.dim() != 1 || t.size(0) != B || t.scalar_type() != at::kInt) refuse(what, name, " must be int32 [", B, "]");
  contiguous(name, t);
}

std::tuple<Tensor, Tensor> step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                                const Tensor& parents, const Tensor& state, double scale, at::ScalarType out_dtype,
                                const OptTensor& out, const OptTensor& u_out) {
  const char* what = "kda_tree_step";
  if (q.dim() != 4 || k.sizes() != q.sizes() || g.sizes() != q.sizes()) refuse(what, "q, k, g must share a [B,N,H,dk] shape");
  const int64_t B = q.size(0), N = q.size(1), H = q.size(2), dk = q.size(3);
  if (v.dim() != 4 || v.size(0) != B || v.size(1) != N || v.size(2) != H) refuse(what, "v must be [B,N,H,dv]");
  const int64_t dv = v.size(3);
  if (beta.dim() != 3 || beta.size(0) != B || beta.size(1) != N || beta.size(2) != H) refuse(what, "beta must be [B,N,H]");
  const int code = code_of(q);
  if (code < 0) refuse(what, "q, k, v, g, beta must share a dtype in bf16/fp16/fp32");
  for (const Tensor* t : {&k, &v, &g, &beta})
    if (t->scalar_type() != q.scalar_type()) refuse(what, "q, k, v, g, beta must share a dtype in bf16/fp16/fp32");
  if (std::max({B, N, H, dk, dv}) > INT32_MAX) refuse(what, "sizes past 2^31");
  places(what, parents, B, N);
  if (state.scalar_type() != at::kFloat || state.dim() != 4 || state.size(0) != B || state.size(1) != H || state.size(2) != dk ||
      state.size(3) != dv)
    refuse(what, "state must be fp32 [", B, ", ", H, ", ", dk, ", ", dv, "]");
  if (out_dtype != at::kFloat && out_dtype != at::kBFloat16) refuse(what, "out_dtype must be fp32 or bf16");
  contiguous("q", q); contiguous("k", k); contiguous("v", v); contiguous("g", g); contiguous("beta", beta); contiguous("state", state);
  const at::Device d = one_gpu(what, q, k, v, g, beta, parents, state);
  const c10::DeviceGuard on(d);
  Tensor o = output(what, "out", out, {B, N, H, dv}, out_dtype, d);
  Tensor u = output(what, "u", u_out, {B, N, H, dv}, at::kFloat, d);
  checked(kda_tree_step(stream_of(d), ptr(q), ptr(k), ptr(v), ptr(g), ptr(beta), i32(parents), static_cast<const float*>(ptr(state)),
                        ptr(o), static_cast<float*>(ptr(u)), B, N, H, dk, dv, static_cast<float>(scale), code,
                        out_dtype == at::kFloat ? KDA_DTYPE_F32 : KDA_DTYPE_BF16),
          what);
  written(out);
  written(u_out);
  return {o, u};
}

Tensor commit(const Tensor& k, const Tensor& g, const Tensor& u, const Tensor& parents, const Tensor& last, Tensor state) {
  const char* what = "kda_tree_commit";
  if (k.dim() != 4 || g.sizes() != k.sizes()) refuse(what, "k, g must share a [B,N,H,dk] shape");
  const int64_t B = k.size(0), N = k.size(1), H = k.size(2), dk = k.size(3);
  if (u.dim() != 4 || u.size(0) != B || u.size(1) != N || u.size(2) != H || u.scalar_type() != at::kFloat)
    refuse(what, "u must be fp32 [B,N,H,dv]");
  const int64_t dv = u.size(3);
  const int code = code_of(k);
  if (code < 0 || g.scalar_type() != k.scalar_type()) refuse(what, "k, g must share a dtype in bf16/fp16/fp32");
  if (std::max({B, N, H, dk, dv}) > INT32_MAX) refuse(what, "sizes past 2^31");
  places(what, parents, B, N);
  per_sequence(what, "last", last, B);
  if (state.scalar_type() != at::kFloat || state.dim() != 4 || state.size(0) != B || state.size(1) != H || state.size(2) != dk ||
      state.size(3) != dv)
    refuse(what, "state must be fp32 [", B, ", ", H, ", ", dk, ", ", dv, "]");
  contiguous("k", k); contiguous("g", g); contiguous("u", u); contiguous("state", state);
  const at::Device d = one_gpu(what, k, g, u, parents, last, state);
  const c10::DeviceGuard on(d);
  checked(kda_tree_commit(stream_of(d), ptr(k), ptr(g), static_cast<const float*>(ptr(u)), i32(parents), i32(last),
                          static_cast<float*>(ptr(state)), B, N, H, dk, dv, code),
          what);
  written(state);
  return state;
}

// sizes of a paged cache and its block table, of `layers` caches behind each other
struct Paged { int64_t layers, pages; int page, per, R, dr, code; };
Paged paged(const char* what, const Tensor& cache, const Tensor& table, const Tensor& lens, int64_t B, bool stacked) {
  const int64_t n = cache.dim();
  if (n != 3 && !(stacked && n == 4)) refuse(what, "cache must be ", stacked ? "[(layers,) n_pages, page_size, R+dr]" : "[n_pages, page_size, R+dr]");
  const int64_t W = cache.size(n - 1), R = W > 512 ? 512 : 256;
  Paged p;
  p.code = code_of(cache);
  if (p.code < 0) refuse(what, "cache must be bf16, fp16 or fp32");
  if (table.dim() != 2 || table.size(0) != B || table.scalar_type() != at::kInt) refuse(what, "block_table must be int32 [", B, ", max_pages]");
  if (std::max({B, W, cache.size(n - 2), table.size(1), n == 4 ? cache.size(0) : 1}) > INT32_MAX) refuse(what, "sizes past 2^31");
  per_sequence(what, "seq_lens", lens, B);
  contiguous("cache", cache);
  contiguous("block_table", table);
  p.layers = n == 4 ? cache.size(0) : 1;
  p.pages = cache.size(n - 3);
  p.page = cache.size(n - 2);
  p.per = table.size(1);
  p.R = R;
  p.dr = W - R;
  return p;
}

std::tuple<Tensor, Tensor> tree_decode(const Tensor& q, const Tensor& cache, const Tensor& table, const Tensor& lens,
                                       const Tensor& parents, double scale, const OptTensor& out, const OptTensor& lse_out,
                                       const OptTensor& workspace) {
  const char* what = "latent_tree_decode";
  if (q.dim() != 4 || cache.dim() != 3 || q.size(3) != cache.size(2))
    refuse(what, "q must be [B,N,H,R+dr] and cache [n_pages, page_size, R+dr]");
  const int64_t B = q.size(0), N = q.size(1), H = q.size(2);
  const Paged p = paged(what, cache, table, lens, B, false);
  if (q.scalar_type() != cache.scalar_type()) refuse(what, "q and cache must share a dtype in bf16/fp16/fp32");
  if (H > INT32_MAX) refuse(what, "sizes past 2^31");
  places(what, parents, B, N);
  contiguous("q", q);
  const at::Device d = one_gpu(what, q, cache, table, lens, parents);
  const c10::DeviceGuard on(d);
  const size_t bytes = kda_latent_tree_decode_workspace(B, N, H, p.R, p.dr, p.page, p.per, p.code);
  const Tensor ws = work(workspace, bytes, d);
  Tensor o = output(what, "out", out, {B, N, H, p.R}, q.scalar_type(), d);
  Tensor lse = output(what, "lse", lse_out, {B, N, H}, at::kFloat, d);
  checked(kda_latent_tree_decode(stream_of(d), ptr(q), ptr(cache), i32(table), i32(lens), i32(parents), ptr(o),
                                 static_cast<float*>(ptr(lse)), B, N, H, p.R, p.dr, p.pages, p.page, p.per, static_cast<float>(scale),
                                 p.code, work_ptr(ws), bytes),
          what);
  written(out);
  written(lse_out);
  return {o, lse};
}

Tensor cache_commit(Tensor cache, const Tensor& table, const Tensor& lens, const Tensor& parents, const Tensor& last, const OptTensor& out) {
  const char* what = "latent_tree_commit";
  if (parents.dim() != 2) refuse(what, "parents must be int32 [B, N]");
  const int64_t B = parents.size(0), N = parents.size(1);
  const Paged p = paged(what, cache, table, lens, B, true);
  places(what, parents, B, N);
  per_sequence(what, "last", last, B);
  if (p.layers < 1) refuse(what, "cache has no layers");
  const at::Device d = one_gpu(what, cache, table, lens, parents, last);
  const c10::DeviceGuard on(d);
  Tensor new_lens = output(what, "out", out, {B}, at::kInt, d);
  checked(kda_latent_tree_commit(stream_of(d), ptr(cache), i32(table), i32(lens), i32(parents), i32(last),
                                 static_cast<int32_t*>(ptr(new_lens)), p.layers, B, N, p.R, p.dr, p.pages, p.page, p.per, p.code),
          what);
  written(cache);
  written(out);
  return new_lens;
}

std::tuple<Tensor, Tensor, Tensor> verify(const Tensor& target, const Tensor& tokens, const Tensor& parents, const OptTensor& uniforms,
                                          const OptTensor& draft, const OptTensor& workspace) {
  const char* what = "tree_verify";
  if (target.dim() != 3 || target.size(1) < 2 || target.size(2) < 1) refuse(what, "target must be [B, N+1, V]");
  const int64_t B = target.size(0), N = target.size(1) - 1, V = target.size(2);
  const int code = code_of(target);
  if (code < 0) refuse(what, "target must be bf16, fp16 or fp32");
  if (std::max(B, V) > INT32_MAX) refuse(what, "sizes past 2^31");
  if (V > 1 && target.stride(2) != 1) refuse(what, "the last axis of target must be contiguous");
  places(what, parents, B, N);
  if (tokens.dim() != 2 || tokens.size(0) != B || tokens.size(1) != N || tokens.scalar_type() != at::kLong)
    refuse(what, "tokens must be int64 [", B, ", ", N, "]");
  contiguous("tokens", tokens);
  if (uniforms) {
    if (uniforms->dim() != 2 || uniforms->size(0) != B || uniforms->size(1) != N + 1 || uniforms->scalar_type() != at::kFloat)
      refuse(what, "uniforms must be fp32 [", B, ", ", N + 1, "]");
    contiguous("uniforms", *uniforms);
  }
  int64_t d_b = 0, d_row = 0;
  if (draft) {
    if (!uniforms) refuse(what, "draft requires uniforms");
    if (draft->dim() != 3 || draft->size(0) != B || draft->size(1) != N || draft->size(2) != V || draft->scalar_type() != target.scalar_type())
      refuse(what, "draft must be ", target.scalar_type(), " [", B, ", ", N, ", ", V, "]");
    if (V > 1 && draft->stride(2) != 1) refuse(what, "the last axis of draft must be contiguous");
    d_b = draft->stride(0);
    d_row = draft->stride(1);
  }
  const at::Device d = one_gpu(what, target, tokens, parents, uniforms, draft);
  const c10::DeviceGuard on(d);
  const size_t bytes = kda_tree_verify_workspace(B, N, V);
  const Tensor ws = work(workspace, bytes, d);
  const auto opt = at::TensorOptions().device(d);
  Tensor last = at::empty({B}, opt.dtype(at::kInt)), next = at::empty({B}, opt.dtype(at::kLong)), accepted = at::empty({B}, opt.dtype(at::kInt));
  checked(kda_tree_verify(stream_of(d), ptr(target), target.stride(0), target.stride(1), static_cast<const int64_t*>(ptr(tokens)),
                          i32(parents), static_cast<const float*>(ptr(uniforms)), ptr(draft), d_b, d_row,
                          static_cast<int32_t*>(ptr(last)), static_cast<int64_t*>(ptr(next)), static_cast<int32_t*>(ptr(accepted)), B, N,
                          V, code, work_ptr(ws), bytes),
          what);
  return {last, next, accepted};
}

}  // namespace

void bind_tree(py::module_& m) {
  m.def("tree_step", &step);
  m.def("tree_commit", &commit);
  m.def("tree_decode", &tree_decode);
  m.def("tree_cache_commit", &cache_commit);
  m.def("tree_verify", &verify);
}
