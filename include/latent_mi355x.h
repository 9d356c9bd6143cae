/*
 * latent_mi355x.h -- C ABI of the latent attention of the MI355X (gfx950) KDA
 * library: the same library file, status codes, dtypes, conventions (device
 * pointers, caller's stream, nothing allocated, arguments rejected before
 * anything is enqueued) and kda_last_error() as kda_mi355x.h.
 */
#ifndef LATENT_MI355X_H_
#define LATENT_MI355X_H_

#include "kda_mi355x.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Latent attention: the softmax layers that stand between KDA layers (the
 * reference's backbone has one to three of them, net/mla.py).  One latent
 * vector of R elements and one rotated key part of dr elements a token are all
 * that a program keeps; every head's keys and values come from the latent.
 *
 * kda_latent_attn_fwd is the expanded form, for prompts and training: per
 * head h, with q = (q_n | q_r), kv = (k_n | v) the up-projection's output as
 * it is, and the rotary key k_r shared by all heads,
 *   s_ij = scale (q_n,i . k_n,j + q_r,i . k_r,j),  o_i = sum_j softmax_j(s_i) v_j,
 *   lse_i = log sum_j exp(s_ij)  (natural logarithm).
 * q [B,Tq,H,dn+dr], kv [B,Tk,H,2 dn], k_rope [B,Tk,dr] in dtype (F32, BF16 or
 * F16), their last axis contiguous and the others by `strides`, a host array
 * of eight element strides: q's (batch, token, head), kv's (batch, token,
 * head), k_rope's (batch, token).  o [B,Tq,H,dn] in dtype, contiguous; lse
 * [B,H,Tq] fp32.  causal != 0: query i sees keys j <= i + Tk - Tq (the last
 * query sees all).  A query that sees no key gets o = 0 and lse = -inf (dq = 0),
 * whatever the keys hold.  Else a masked pair enters the products of its tile
 * with weight 0: values that are not finite in a key, query or cotangent may
 * reach rows of the same sequence that do not see them, never those of another
 * batch element or packed sequence.
 * cu_q, cu_k (both or neither; int32 [n_seqs+1] on the device, B == 1) pack
 * n_seqs sequences, sequence i being rows cu[i] .. cu[i+1] of its axis; the
 * first offset is 0 and the last the axis' length.  Offsets are clamped so
 * that no access leaves the tensors; malformed ones leave rows unwritten.
 * dn in {64, 128}, dr in {32, 64}, scale > 0 and finite, Tq, Tk >= 0.
 * Products run in the inputs' precision (probabilities rounded to it for the
 * second), sums and softmax statistics in fp32.  Pointers are aligned to 16
 * bytes and strides are multiples of 16 bytes.  Calls of few blocks of 128
 * queries share each block's keys out over workgroups and join their parts:
 * caller workspace of kda_latent_attn_fwd_workspace bytes.
 */
KDA_API int kda_latent_attn_fwd(hipStream_t stream, const void* q, const void* kv, const void* k_rope,
                const int64_t* strides, const int32_t* cu_q, const int32_t* cu_k, int32_t n_seqs,
                void* o, float* lse, int B, int Tq, int Tk, int H, int dn, int dr, int causal, float scale,
                int dtype, void* workspace, size_t workspace_bytes);

/* Workspace bytes kda_latent_attn_fwd needs (n_seqs 0: dense).  0 where it
 * needs none (enough blocks of 128 queries to fill the chip; also on bad
 * input): then workspace may be null.  Host-only. */
KDA_API size_t kda_latent_attn_fwd_workspace(int B, int Tq, int Tk, int H, int dn, int dr, int32_t n_seqs, int dtype);

/*
 * Gradients of o of kda_latent_attn_fwd: given its inputs, o, lse and the
 * cotangent d_o [B,Tq,H,dn] (dtype, contiguous), writes dq [B,Tq,H,dn+dr],
 * dkv [B,Tk,H,2 dn] and dk_rope [B,Tk,dr] (summed over the heads), contiguous,
 * in dtype, rounded once from fp32 sums.  No atomics: the same bits in every
 * run.  Caller workspace of kda_latent_attn_bwd_workspace bytes.
 */
KDA_API int kda_latent_attn_bwd(hipStream_t stream, const void* q, const void* kv, const void* k_rope,
                const int64_t* strides, const int32_t* cu_q, const int32_t* cu_k, int32_t n_seqs,
                const void* o, const float* lse, const void* d_o, void* dq, void* dkv, void* dk_rope,
                int B, int Tq, int Tk, int H, int dn, int dr, int causal, float scale, int dtype,
                void* workspace, size_t workspace_bytes);

/* Workspace bytes kda_latent_attn_bwd needs (n_seqs 0: dense; 0 on bad input).  Host-only. */
KDA_API size_t kda_latent_attn_bwd_workspace(int B, int Tq, int Tk, int H, int dn, int dr, int32_t n_seqs, int dtype);

/*
 * New tokens into the latent cache: row i of `rows` [N, R+dr] (the
 * down-projection's output; element stride rows_stride) gets its first R
 * elements normed, x / sqrt(mean x^2 + eps) * norm_weight (fp32 [R]; null:
 * taken as they are), its last dr elements rotated by the angles of position
 * positions[i] (int64), and is stored at row slots[i] (int64; page *
 * page_size + offset) of cache [n_slots, R+dr].  A slot outside [0, n_slots)
 * is not stored (padding rows).  cos_sin [n_positions, dr] fp32 holds the
 * cosines of the dr/2 angles of a position and then their sines; a position
 * outside it takes the nearest row.  interleaved == 0: element i pairs with i
 * + dr/2; else 2i with 2i + 1.  In the same launch the queries' rotary parts
 * q [N, H, dr] (null: none; strides in elements) are rotated into q_out
 * (which may be q).  R in {256, 512}, dr in {32, 64}, N >= 0.  rows, cache,
 * cos_sin and norm_weight are aligned to 16 bytes (rows_stride too), q and
 * q_out with their strides to 4 elements.
 */
KDA_API int kda_latent_append(hipStream_t stream, const void* rows, int64_t rows_stride, const int64_t* positions,
                const int64_t* slots, const float* cos_sin, int64_t n_positions, const float* norm_weight, float eps,
                void* cache, int64_t n_slots, const void* q, int64_t q_stride_t, int64_t q_stride_h, void* q_out,
                int64_t qo_stride_t, int64_t qo_stride_h, int N, int H, int R, int dr, int interleaved, int dtype);

/*
 * Latent attention over the paged cache (absorbed form), for one to a few
 * tokens of every sequence: q [B,Tq,H,R+dr] (the nope query times the
 * key up-projection, R elements, then the rotated part), cache
 * [n_pages, page_size, R+dr], block_table int32 [B, max_pages] (the pages of a
 * sequence in order), seq_lens int32 [B] (tokens in the cache, the Tq new
 * ones among them):
 *   s_j = scale q . row_j,  o = sum_j softmax_j(s) row_j[:R],  lse as above.
 * Token t sees the first seq_len - (Tq - 1 - t) rows; with none, o = 0 and
 * lse = -inf, whatever the rows hold (else a row of the newest Tq that is not
 * finite may reach the earlier tokens of its sequence).  o [B,Tq,H,R] in dtype, lse [B,Tq,H] fp32; all contiguous.
 * Lengths are clamped into [0, max_pages * page_size] and page numbers into
 * [0, n_pages), so no access leaves the tensors.  R in {256, 512}, dr in {32,
 * 64}, page_size a power of two, n_pages * page_size < 2^31, scale > 0 and
 * finite.  Two launches: the sequences' key tiles in equal runs over the
 * chip, then the join of sequences that more than one run covered.  Caller
 * workspace of kda_latent_decode_workspace bytes.  Pointers aligned to 16
 * bytes.
 */
KDA_API int kda_latent_decode(hipStream_t stream, const void* q, const void* cache, const int32_t* block_table,
                const int32_t* seq_lens, void* o, float* lse, int B, int Tq, int H, int R, int dr, int64_t n_pages,
                int page_size, int max_pages, float scale, int dtype, void* workspace, size_t workspace_bytes);

/* Workspace bytes kda_latent_decode needs (0 on bad input).  Host-only. */
KDA_API size_t kda_latent_decode_workspace(int B, int Tq, int H, int R, int dr, int page_size, int max_pages, int dtype);

#ifdef __cplusplus
}
#endif

#endif /* LATENT_MI355X_H_ */
