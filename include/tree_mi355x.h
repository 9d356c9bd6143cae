/*
 * tree_mi355x.h -- C ABI of the tree calls of the MI355X (gfx950) KDA library:
 * a tree of drafted tokens looked at in one step, over KDA states and the
 * latent cache.  The same library file, status codes, dtypes, conventions
 * (device pointers, caller's stream, nothing allocated, arguments rejected
 * before anything is enqueued) and kda_last_error() as kda_mi355x.h.
 *
 * Trees.  A sequence has N places (1 <= N <= 64) for drafted tokens; parents
 * int32 [B,N] holds, for place i, the place in [0, i) that it continues, or -1
 * if it continues the sequence itself.  Any other entry marks a place that
 * holds no draft; a place below such a one holds none either.  The path of
 * place i: its ancestors and itself, in the order of their indices.  Trees are
 * read on the device; every value of parents is safe.  Places without a
 * draft get zeros, and what their inputs hold reaches nothing.  A draft
 * whose own values are not finite may reach other drafts of its sequence and
 * head, on its path or not.  What a call writes must not overlap its other
 * arguments.
 */
#ifndef TREE_MI355X_H_
#define TREE_MI355X_H_

#include "latent_mi355x.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * kda_recurrent_step over a tree, the state left as it is: q, k, g [B,N,H,dk],
 * v [B,N,H,dv], beta [B,N,H] in in_dtype (F32, BF16 or F16), state [B,H,dk,dv]
 * fp32, everything contiguous.  With a_i = exp(g_i), S the state after the
 * parent of i (`state` itself for -1):
 *   S~ = diag(a_i) S,  u_i = beta_i (v_i - S~^T k_i),  S_i = S~ + k_i u_i^T,
 *   o_i = scale S_i^T q_i.
 * o [B,N,H,dv] in out_dtype (F32 or BF16); u [B,N,H,dv] fp32, what
 * kda_tree_commit needs of the call.  dk == dv in {64, 128}.  Pointers aligned
 * to 16 bytes (beta and parents to their elements).  A decay between two places is
 * as exact as those of the places between them, however far the path has decayed
 * before.  In the read-out of `state` the bits of scale q_i and k_i times their
 * path's decay end at 2^-126, and so do those of a state's entries beside ones of
 * 2^-63 and more.
 */
KDA_API int kda_tree_step(hipStream_t stream, const void* q, const void* k, const void* v, const void* g,
                const void* beta, const int32_t* parents, const float* state, void* o, float* u, int B, int N, int H,
                int dk, int dv, float scale, int in_dtype, int out_dtype);

/*
 * The state after the path of place last[b] (int32 [B]), in place: state
 * [B,H,dk,dv] goes from before the tree to S_last, from the k, g (in_dtype)
 * and u of the kda_tree_step call.  last[b] outside [0, N), or a place without
 * a draft: the state is left as it is.
 */
KDA_API int kda_tree_commit(hipStream_t stream, const void* k, const void* g, const float* u, const int32_t* parents,
                const int32_t* last, float* state, int B, int N, int H, int dk, int dv, int in_dtype);

/*
 * kda_latent_decode over a tree: q [B,N,H,R+dr] and the rows of the N places
 * are the newest of the sequence, place i in row seq_len - N + i of its pages
 * (a place without a draft has a row too; what it holds is not read).  Place i
 * sees the rows before those of the places, and those of its path:
 *   s_j = scale q . row_j,  o = sum_j softmax_j(s) row_j[:R],  lse natural.
 * Places without a draft, and those whose row would lie before the sequence's
 * first (seq_len < N), get o = 0 and lse = -inf.  The rest as
 * kda_latent_decode: o [B,N,H,R] in dtype, lse [B,N,H] fp32, page numbers and
 * lengths clamped, R in {256, 512}, dr in {32, 64}, page_size a power of two,
 * caller workspace of kda_latent_tree_decode_workspace bytes, pointers aligned
 * to 16 bytes (tables to their elements).
 */
KDA_API int kda_latent_tree_decode(hipStream_t stream, const void* q, const void* cache, const int32_t* block_table,
                const int32_t* seq_lens, const int32_t* parents, void* o, float* lse, int B, int N, int H, int R, int dr,
                int64_t n_pages, int page_size, int max_pages, float scale, int dtype, void* workspace,
                size_t workspace_bytes);

/* Workspace bytes kda_latent_tree_decode needs (0 on bad input).  Host-only. */
KDA_API size_t kda_latent_tree_decode_workspace(int B, int N, int H, int R, int dr, int page_size, int max_pages, int dtype);

/*
 * The cache after the path of place last[b]: of the N newest rows of a
 * sequence, those of the path move to the front, in order (place path[i] from
 * row seq_len - N + path[i] to row seq_len - N + i), in each of the `layers`
 * caches [n_pages, page_size, R+dr] that lie one behind the other and share
 * the block table; new_lens[b] = seq_len - N + the path's length.  last[b]
 * outside [0, N), or a place without a draft: the path is empty.  A sequence
 * of fewer than N rows is left as it is, its length too.  new_lens is not
 * seq_lens, which calls for further layers still read.  Page numbers and lengths are clamped as in
 * kda_latent_tree_decode.  cache aligned to 16 bytes.
 */
KDA_API int kda_latent_tree_commit(hipStream_t stream, void* cache, const int32_t* block_table, const int32_t* seq_lens,
                const int32_t* parents, const int32_t* last, int32_t* new_lens, int layers, int B, int N, int R, int dr,
                int64_t n_pages, int page_size, int max_pages, int dtype);

/*
 * Which path the target accepts.  target [B,N+1,V] in dtype (F32, BF16 or
 * F16): row 0 belongs to the sequence's end, row i + 1 to place i; tokens
 * int64 [B,N]; V contiguous, the other axes by element strides.
 *
 * uniforms null: target holds scores of any kind.  At row r the token is
 * argmax (the lowest index where several are largest; NaN is never the
 * largest; 0 where all are NaN); the walk goes from the sequence to the first
 * child whose token it is, and on.
 *
 * uniforms fp32 [B,N+1] in [0, 1): target holds finite probabilities.  At a row the
 * children are asked in the order of their indices; with R the row and Z = 1
 * at first, child i of token x is accepted if uniforms[i] q_i(x) Z < R(x).
 * If not, R becomes max(R - Z q_i, 0) and Z its sum, and the next is asked.
 * q_i: draft[i], the distribution that the token was drawn from ([B,N,V] in
 * dtype; null: a token chosen without chance, q_i(x) = 1 and 0 elsewhere,
 * where R(x) becomes 0 and Z loses R(x)).  When no child is left the next
 * token is drawn from R: the lowest v whose running sum is over uniforms[N]
 * times the whole sum (where R has none, from the row as it was; -1 where
 * that has none; entries that are not positive count as 0).  So the accepted
 * tokens and the next are distributed as the target's own draws.  Sums,
 * products and comparisons in 64 bits.  With draft the k-th refusal at a row
 * reads k + 1 rows of V again: many refused children of one place are slow.  A token outside [0, V) is never
 * accepted.
 *
 * last int32 [B]: the last accepted place (-1: none); next int64 [B]: the
 * token that follows; accepted int32 [B]: how many places the path has.
 * Caller workspace of kda_tree_verify_workspace bytes, aligned to 16 bytes.
 */
KDA_API int kda_tree_verify(hipStream_t stream, const void* target, int64_t target_b, int64_t target_row,
                const int64_t* tokens, const int32_t* parents, const float* uniforms, const void* draft,
                int64_t draft_b, int64_t draft_row, int32_t* last, int64_t* next, int32_t* accepted, int B, int N, int V,
                int dtype, void* workspace, size_t workspace_bytes);

/* Workspace bytes kda_tree_verify needs, for every mode (0 on bad input).  Host-only. */
KDA_API size_t kda_tree_verify_workspace(int B, int N, int V);

#ifdef __cplusplus
}
#endif

#endif /* TREE_MI355X_H_ */
