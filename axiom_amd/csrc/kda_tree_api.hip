// C ABI of the tree calls on KDA states and of the verification: argument validation, plans, dispatch
// (the latent ones: kda_latent_api.hip).
#include "tree_mi355x.h"

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <initializer_list>

#include "kda_internal.h"

namespace {

int fail(int code, const char* fmt, ...) {
  char msg[400];
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  return kda::api_fail(code, msg);
}
int launched(hipError_t e, const char* what) {
  return e == hipSuccess ? KDA_OK : fail(KDA_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}
bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
size_t elem(int dtype) { return dtype == KDA_DTYPE_F32 ? 4 : 2; }
bool dtype_ok(int dtype) { return dtype == KDA_DTYPE_F32 || dtype == KDA_DTYPE_BF16 || dtype == KDA_DTYPE_F16; }

constexpr int kPlaces = 64;
constexpr int64_t kMaxBlocks = int64_t{1} << 22;   // 1024 threads each

int check_states(int B, int N, int H, int dk, int dv, int dtype) {
  if (!dtype_ok(dtype)) return fail(KDA_ERR_INVALID_ARGUMENT, "in_dtype=%d must be F32, BF16 or F16", dtype);
  if (B < 0 || N < 1 || H < 1) return fail(KDA_ERR_INVALID_ARGUMENT, "sizes B=%d N=%d H=%d out of range", B, N, H);
  if (N > kPlaces) return fail(KDA_ERR_UNSUPPORTED, "N=%d places, %d at most", N, kPlaces);
  if (dk != dv || (dk != 64 && dk != 128)) return fail(KDA_ERR_UNSUPPORTED, "head dims dk=%d, dv=%d unsupported (dk == dv in {64, 128})", dk, dv);
  if (static_cast<int64_t>(B) * H > kMaxBlocks) return fail(KDA_ERR_UNSUPPORTED, "B * H = %lld too large", static_cast<long long>(B) * H);
  return KDA_OK;
}

// Slices of a row, a workgroup each.  Drawing: one workgroup a CU over all
// sequences, none under 4096 entries (a wave's share is then one round of loads); greedy, where all
// rows of all sequences are looked at: four, none under 2048.
int draw_slices(int64_t B, int64_t V) {
  return static_cast<int>(std::max<int64_t>(1, std::min({int64_t{64}, 256 / std::max<int64_t>(B, 1), V / 4096})));
}
int greedy_slices(int64_t rows, int64_t V) {
  return static_cast<int>(std::max<int64_t>(1, std::min({int64_t{64}, 1024 / std::max<int64_t>(rows, 1), V / 2048})));
}
constexpr size_t kWalkBytes = 16 + 8 * kPlaces, kPieceBytes = 16 * 16;   // a sequence's walk; a slice's sums

}  // namespace

extern "C" {

int kda_tree_step(hipStream_t stream, const void* q, const void* k, const void* v, const void* g, const void* beta,
                  const int32_t* parents, const float* state, void* o, float* u, int B, int N, int H, int dk, int dv,
                  float scale, int in_dtype, int out_dtype) {
  if (const int rc = check_states(B, N, H, dk, dv, in_dtype)) return rc;
  if (out_dtype != KDA_DTYPE_F32 && out_dtype != KDA_DTYPE_BF16)
    return fail(KDA_ERR_INVALID_ARGUMENT, "out_dtype=%d: o is emitted as F32 or BF16", out_dtype);
  if (!std::isfinite(scale)) return fail(KDA_ERR_INVALID_ARGUMENT, "scale must be finite");
  if (B == 0) return KDA_OK;
  if (!q || !k || !v || !g || !beta || !parents || !state || !o || !u) return fail(KDA_ERR_INVALID_ARGUMENT, "null pointer");
  for (const void* p : {q, k, v, g, static_cast<const void*>(state), static_cast<const void*>(o), static_cast<const void*>(u)})
    if (!aligned(p, 16)) return fail(KDA_ERR_INVALID_ARGUMENT, "q, k, v, g, state, o and u must be aligned to 16 bytes");
  const size_t bn = static_cast<size_t>(B) * N, rows = bn * H, in = rows * dk * elem(in_dtype);
  if (kda::overlap({{o, rows * dv * elem(out_dtype)}, {u, rows * dv * 4}},
                   {{q, in}, {k, in}, {v, in}, {g, in}, {beta, rows * elem(in_dtype)}, {parents, bn * 4},
                    {state, static_cast<size_t>(B) * H * dk * dv * 4}}))
    return fail(KDA_ERR_INVALID_ARGUMENT, "o and u must not overlap each other or the inputs");
  kda::TreeStepArgs a{};
  a.q = q; a.k = k; a.v = v; a.g = g; a.beta = beta; a.parents = parents; a.state = state; a.o = o; a.u = u;
  a.B = B; a.N = N; a.H = H; a.scale = scale;
  return launched(kda::launch_tree_step(a, dk, in_dtype, out_dtype == KDA_DTYPE_BF16 ? 1 : 0, stream), "kda_tree_step");
}

int kda_tree_commit(hipStream_t stream, const void* k, const void* g, const float* u, const int32_t* parents, const int32_t* last,
                    float* state, int B, int N, int H, int dk, int dv, int in_dtype) {
  if (const int rc = check_states(B, N, H, dk, dv, in_dtype)) return rc;
  if (B == 0) return KDA_OK;
  if (!k || !g || !u || !parents || !last || !state) return fail(KDA_ERR_INVALID_ARGUMENT, "null pointer");
  for (const void* p : {k, g, static_cast<const void*>(u), static_cast<const void*>(state)})
    if (!aligned(p, 16)) return fail(KDA_ERR_INVALID_ARGUMENT, "k, g, u and state must be aligned to 16 bytes");
  const size_t bn = static_cast<size_t>(B) * N, rows = bn * H, in = rows * dk * elem(in_dtype);
  if (kda::overlap({{state, static_cast<size_t>(B) * H * dk * dv * 4}},
                   {{k, in}, {g, in}, {u, rows * dv * 4}, {parents, bn * 4}, {last, static_cast<size_t>(B) * 4}}))
    return fail(KDA_ERR_INVALID_ARGUMENT, "state must not overlap the other arguments");
  kda::TreeCommitArgs a{};
  a.k = k; a.g = g; a.u = u; a.parents = parents; a.last = last; a.state = state;
  a.B = B; a.N = N; a.H = H;
  return launched(kda::launch_tree_commit(a, dk, in_dtype, stream), "kda_tree_commit");
}

size_t kda_tree_verify_workspace(int B, int N, int V) {
  if (B < 0 || N < 1 || N > kPlaces || V < 1) return 0;
  const size_t rows = static_cast<size_t>(B) * (N + 1);
  return std::max({static_cast<size_t>(B) * (kWalkBytes + draw_slices(B, V) * kPieceBytes),
                   rows * greedy_slices(static_cast<int64_t>(rows), V) * 8, size_t{16}});
}

int kda_tree_verify(hipStream_t stream, const void* target, int64_t target_b, int64_t target_row, const int64_t* tokens,
                    const int32_t* parents, const float* uniforms, const void* draft, int64_t draft_b, int64_t draft_row,
                    int32_t* last, int64_t* next, int32_t* accepted, int B, int N, int V, int dtype, void* workspace,
                    size_t workspace_bytes) {
  if (!dtype_ok(dtype)) return fail(KDA_ERR_INVALID_ARGUMENT, "dtype=%d must be F32, BF16 or F16", dtype);
  if (B < 0 || N < 1 || V < 1) return fail(KDA_ERR_INVALID_ARGUMENT, "sizes B=%d N=%d V=%d out of range", B, N, V);
  if (N > kPlaces) return fail(KDA_ERR_UNSUPPORTED, "N=%d places, %d at most", N, kPlaces);
  if (V > (1 << 30)) return fail(KDA_ERR_UNSUPPORTED, "V=%d over 2^30", V);
  const int64_t rows = static_cast<int64_t>(B) * (N + 1);
  if (rows > kMaxBlocks) return fail(KDA_ERR_UNSUPPORTED, "B * (N + 1) = %lld too large", static_cast<long long>(rows));
  if (target_b < 0 || target_row < 0 || draft_b < 0 || draft_row < 0) return fail(KDA_ERR_INVALID_ARGUMENT, "strides must not be negative");
  if (draft && !uniforms) return fail(KDA_ERR_INVALID_ARGUMENT, "draft goes with uniforms");
  if (B == 0) return KDA_OK;
  if (!target || !tokens || !parents || !last || !next || !accepted) return fail(KDA_ERR_INVALID_ARGUMENT, "null pointer");
  if (!workspace || workspace_bytes < kda_tree_verify_workspace(B, N, V))
    return fail(KDA_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : size_t{0},
                kda_tree_verify_workspace(B, N, V));
  if (!aligned(workspace, 16)) return fail(KDA_ERR_INVALID_ARGUMENT, "workspace must be aligned to 16 bytes");
  auto extent = [&](int64_t s_b, int64_t s_row, int n) {   // of n rows a sequence
    return static_cast<size_t>((B - 1) * s_b + (n - 1) * s_row + V) * elem(dtype);
  };
  const size_t b4 = static_cast<size_t>(B) * 4, bn = static_cast<size_t>(B) * N;
  if (kda::overlap({{last, b4}, {next, 2 * b4}, {accepted, b4}, {workspace, kda_tree_verify_workspace(B, N, V)}},
                   {{target, extent(target_b, target_row, N + 1)}, {tokens, bn * 8}, {parents, bn * 4}, {uniforms, (bn + B) * 4},
                    {draft, extent(draft_b, draft_row, N)}}))
    return fail(KDA_ERR_INVALID_ARGUMENT, "last, next, accepted and workspace must not overlap each other or the inputs");
  kda::TreeVerifyArgs a{};
  a.target = target; a.draft = draft; a.tokens = tokens; a.parents = parents; a.uniforms = uniforms;
  a.last = last; a.next = next; a.accepted = accepted;
  a.t_b = target_b; a.t_row = target_row; a.d_b = draft_b; a.d_row = draft_row;
  a.B = B; a.N = N; a.V = V; a.ws = workspace;
  a.slices = uniforms ? draw_slices(B, V) : greedy_slices(rows, V);
  a.per = ((V + a.slices - 1) / a.slices + 63) / 64 * 64;
  return launched(kda::launch_tree_verify(a, dtype, stream), "kda_tree_verify");
}

}  // extern "C"
