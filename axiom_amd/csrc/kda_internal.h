// Internal argument structs and launchers shared by the KDA translation units.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <initializer_list>

namespace kda {

// Geometry of one chunked call.  Dense: B sequences of T tokens (cu == null).
// Varlen: one packed stream of T tokens split by cu_seqlens into N sequences.
struct Geom {
  int B, T, H;
  int NT;                       // dense: chunks per sequence
  int n0;                       // dense: first chunk of the segment this launch covers
  int NTS;                      // dense: chunks in that segment (workspace units per sequence)
  int N;                        // number of sequences (dense: B)
  const int32_t* cu;            // original cu_seqlens (varlen) or null
  const int32_t* cu_clamped;    // validated copy (varlen)
  const int32_t* chunk_off;     // [N+1] first chunk unit of each sequence (varlen)
  const int32_t* n_units;       // total chunk units (varlen, device)
  const int32_t* order;         // longest-first sequence order (varlen) or null
  // Segmented varlen calls (pos_off non-null).  Units are numbered
  // position-major: every sequence's chunk p precedes every sequence's chunk
  // p + 1, and at position p the sequences of longest-first rank 0 ..
  // cnt(p) - 1 (the ones with more than p chunks) hold units pos_off[p] +
  // rank.  A launch covers units [seg * KU, (seg + 1) * KU); its workspace
  // slot of unit u is u - seg * KU.  seg_pos[2 s], seg_pos[2 s + 1] are the
  // position and rank of unit s * KU (the first unit of segment s).
  const int32_t* pos_off;       // [n_pos + 1], device (prep kernel)
  const int32_t* seg_pos;       // [2 (n_seg + 1)], device (prep kernel)
  int seg;                      // segment of this launch
  int KU;                       // units per segment
};

struct IntraArgs {
  Geom geom;
  const void* q;
  const void* k;
  const void* v;
  const void* g;
  const void* beta;
  float scale;
  void* W;    // per chunk-head, fragment order (see kda_chunk.hip)
  void* U;
  void* AQ;
  void* GQ;
  void* LK;
  float* GC;
  // Fused prologue (K > 0): q, k, v are the raw projections qp, kp, vp and
  // the kernel applies the short conv (taps cw[t] [K][H*dk] fp32, history of
  // each sequence's first chunk cb[t] [N][K-1][H*dk] fp32 or null = zeros),
  // swish and, for q and k, the L2 norm before everything else.
  const float* cw[3];
  const float* cb[3];
  int K;
  int* status_clear;   // non-null: the launch zeroes the call's status word
  int total;           // chunk-heads of the launch (overlapped-segment launch only)
  // cc_scan operands (fp32 gates only): g holds alpha (the decay factor; the
  // kernel takes log2(alpha) by the hardware logarithm, the log-decay in the
  // base-2 units it works in) and beta holds beta32 [T*H][32] (the kernel
  // takes the mean of the 32 columns, summed in column order)
  int gates_alpha;
};

struct StateArgs {
  Geom geom;
  const void* W;
  const void* U;
  const void* AQ;
  const void* GQ;
  const void* LK;
  const float* GC;
  const float* h0;
  void* o;
  float* ht;
  // non-null (16-bit inputs): bit kStatusNonFinite is set when an o or final
  // state value of the call is not finite
  int* status;
};

// status word of a chunked forward call: a non-finite o or final state value
// (an fp16 operand out of range, or non-finite inputs)
constexpr int kStatusNonFinite = 1 << 16;

struct DecodeArgs {
  const void* q;
  const void* k;
  const void* v;
  const void* g;
  const void* beta;
  float* state;
  void* o;
  float scale;
};

struct AdaptArgs {
  const float* alpha;
  const float* beta32;
  float* g_out;
  float* beta_out;
  int64_t n_tok_heads;  // T * H
  int dk;
};

// Chunked backward (dense inputs; workspace arrays row-major per chunk-head
// ch = (b * NT + n) * H + h, fp32, or for 16-bit inputs fp16 where kda_bwd.hip
// says so; the F* arrays, written and read only with 16-bit inputs, are fp16
// MFMA A fragments: lane (r = l & 15, gq = l >> 4) of K step s holds M index
// 16 m + r and K indices 32 s + 4 gq + (e & 3) + 16 (e >> 2), e = 0..7).
struct BwdArgs {
  int B, T, H, NT;
  const void* q;
  const void* k;
  const void* v;
  const void* g;
  const void* beta;
  const float* h0;      // [B,H,dk,dv] or null
  const void* dout;     // cotangent of o, [B,T,H,dv] (fp32 or bf16)
  const float* dht;     // cotangent of the final state, [B,H,dk,dv] or null
  float scale;
  void* dq;             // [B,T,H,dk] of element type qkv_out
  void* dk;
  void* dv;             // [B,T,H,dv]
  void* dg;             // [B,T,H,dk] of element type g_out
  void* dbeta;          // [B,T,H]
  int qkv_out, g_out;   // 0 fp32, 1 bf16, 2 fp16 (16-bit only where the input is of that type)
  float* dh0;           // [B,H,dk,dv] or null
  float* QG;            // [ch][C][dk] gamma * q (scaled)
  float* KL;            // [ch][C][dk] lambda * k
  float* GCV;           // [ch][dk]    gamma_C
  float* AQ;            // [ch][C][C]  Aqk
  float* TM;            // [ch][C][C]  (I + L)^-1
  float* WM;            // [ch][C][dk]
  float* UM;            // [ch][C][dv]
  float* SI;            // [ch][dk][dv] state entering the chunk
  float* VT;            // [ch][C][dv] v~
  float* DS;            // [ch][dk][dv] cotangent of the state leaving the chunk
  float* DVT;           // [ch][C][dv] cotangent of v~
  void* FL;             // [ch][4][dk/32][64][8]  lambda k (M rows, K channels)
  void* FA;             // [ch][6][64][8]         Aqk^T (M key rows, K query rows): (key tile, K step)
                        //                        00 01 10 11 21 31 (the others are zero)
  void* FQ;             // [ch][dk/16][2][64][8]  (gamma q)^T (M channels, K rows)
  void* FW;             // [ch][dk/16][2][64][8]  W^T (M channels, K rows)
  void* FWN;            // [ch][4][dk/32][64][8]  W (M rows, K channels)
  void* FLT;            // [ch][dk/16][2][64][8]  (lambda k)^T (M channels, K rows)
};

// Whether two byte ranges share memory (never where one has no address).  Launches
// that were joined keep their order for calls whose outputs lie over their inputs.
inline bool overlaps(const void* p, int64_t pn, const void* q, int64_t qn) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(q);
  return p != nullptr && q != nullptr && x < y + static_cast<uintptr_t>(qn) && y < x + static_cast<uintptr_t>(pn);
}

// Standalone unit-triangular solve (kda_ut.hip); a [H][C][C], b/x/xf [H][C][N].
struct UtArgs {
  const void* a;
  const void* b;    // right-hand side (the cotangent dX in the backward rule)
  void* x;          // solution (dB in the backward rule)
  const void* xf;   // backward rule: the forward solution X
  void* da;         // backward rule: dA (strict lower), else unused
  int H, C, N, ntiles;
};

// Prologue / epilogue around the chunked kernels (kda_prologue.hip).
struct PrologueArgs {
  const void* qp;          // [B,T,H*d] projections (fp32 or bf16)
  const void* kp;
  const void* vp;
  const float* wq;         // [K, H*d] depthwise conv taps, w[i] weights x[t-i]
  const float* wk;
  const float* wv;
  const float* bq_in;      // [B, K-1, H*d] history rows, oldest first, or null (zeros)
  const float* bk_in;
  const float* bv_in;
  float* bq_out;           // last K-1 inputs after this call, or null
  float* bk_out;
  float* bv_out;
  void* q;                 // [B,T,H,d] outputs (fp32 or bf16)
  void* k;
  void* v;
  int B, T, H, K;
};

struct EpilogueArgs {
  const void* o;           // [B,T,H,dv]
  const void* gate;        // [B,T,H*dv] gate logits
  void* y;                 // [B,T,H*dv]
  int B, T, H;
  float eps;
};

// Backward of the prologue: cotangents dq, dk, dv [B,T,H,d] fp32 of its
// outputs -> dx (projections), dw (conv taps), db (incoming buffers).
struct PrologueBwdArgs {
  const void* x[3];        // qp, kp, vp [B,T,H*d] (fp32 or bf16)
  const float* w[3];       // [K, H*d]
  const float* bin[3];     // [B, K-1, H*d] or null (zeros)
  const float* dy[3];      // dq, dk, dv [B,T,H*d] fp32
  void* dx[3];             // [B,T,H*d] fp32, or bf16 with bf16 projections
  float* dw[3];            // [K, H*d] fp32
  float* db[3];            // [B, K-1, H*d] fp32 or null (not wanted)
  float* part;             // workspace: [3][B * G][K][H*d] fp32, dw partial sums (G groups of 64 rows)
  int B, T, H, K, G;
};

struct EpilogueBwdArgs {
  const void* o;           // [B,T,H,dv]
  const void* gate;        // [B,T,H*dv] gate logits
  const void* dy;          // [B,T,H*dv]
  float* dout;             // [B,T,H,dv] fp32
  void* dgate;             // [B,T,H*dv]
  int B, T, H;
  float eps;
};

hipError_t launch_prologue(const PrologueArgs& a, int d, int in_dt, int out_dt, hipStream_t s);
hipError_t launch_prologue_bwd(const PrologueBwdArgs& a, int d, int in_dt, int dx_dt, hipStream_t s);
hipError_t launch_epilogue_bwd(const EpilogueBwdArgs& a, int d, int o_dt, int g_dt, int dy_dt, int dg_dt,
                               hipStream_t s);
// launch_epilogue (fp32 o) and the conv buffer update of launch_prologue (the
// last K-1 inputs; bf16 projections) in one launch
hipError_t launch_epilogue_buffers(const EpilogueArgs& a, const PrologueArgs& p, int d, int g_dt, int y_dt,
                                   hipStream_t s);
hipError_t launch_epilogue(const EpilogueArgs& a, int d, int o_dt, int g_dt, int y_dt, hipStream_t s);
// in_dtype: a kda_dtype_t, or kInAlphaGates (the cc_scan seam: bf16 q, k, v,
// fp32 do; g = alpha, beta = beta32 [token-head][32], dg = dalpha, dbeta =
// dbeta32, bf16 dq, dk, dv)
constexpr int kInAlphaGates = 16;
hipError_t launch_bwd(const BwdArgs& a, int d, int in_dtype, int do_dtype, hipStream_t s);
hipError_t launch_ut(const UtArgs& a, int dtype, bool transpose, bool with_da, hipStream_t s);
// dst[0..n) = src (or 0 when src is null), by a kernel (no memset/memcpy node)
hipError_t launch_copy_or_zero(float* dst, const float* src, int64_t n, hipStream_t s);
hipError_t launch_intra(const IntraArgs& a, int d, int dtq, int dtg, int grid, hipStream_t s);
// the intra kernel with the fused prologue (a.K in [1, kFusedConvTaps], bf16 q, k, v)
hipError_t launch_intra_prologue(const IntraArgs& a, int d, int dtg, int grid, hipStream_t s);
constexpr int kFusedConvTaps = 4;
hipError_t launch_state(const StateArgs& a, int d, bool exact, int out_dt, int grid, hipStream_t s);
// state scan of one segment (n_state workgroups of the 32-column state
// kernel's grid) and intra-chunk work of the next (intra_units chunk-heads)
// in one launch; fp16 operands, no fused prologue
hipError_t launch_overlap(const IntraArgs& ia, const StateArgs& sa, int d, int dtq, int dtg, int out_dt,
                          int n_state, int intra_units, hipStream_t s);
// varlen preparation; pos_off / seg_pos non-null (segmented calls, N <= 2048):
// also the position-major unit tables of Geom for segments of KU units
// (n_seg segments)
hipError_t launch_varlen_prep(const int32_t* cu, int N, int T, int32_t* cu_clamped,
                              int32_t* chunk_off, int32_t* n_units, int32_t* order,
                              int32_t* flags, int32_t* pos_off, int32_t* seg_pos, int KU, int n_seg,
                              hipStream_t s);
hipError_t launch_decode(const DecodeArgs& a, int d, int dt, int out_dt, int grid, hipStream_t s);

// One decode token of the whole layer in one launch: short conv (buffers
// shifted in place), swish, L2 norm of q and k, the delta-rule step on the
// fp32 state in place, head-wise RMSNorm x sigmoid gate.
struct DecodeLayerArgs {
  const void* x[3];        // qp, kp, vp [B, H*d]
  const void* g;           // [B, H, d] log decay
  const void* beta;        // [B, H]
  const void* gate;        // [B, H*d] logits
  const float* w[3];       // conv taps [K, H*d]
  float* buf[3];           // conv buffers [B, K-1, H*d] (updated in place)
  float* state;            // [B, H, d, d]
  void* y;                 // [B, H*d]
  float scale, eps;
  int B, H, K;
};
hipError_t launch_decode_layer(const DecodeLayerArgs& a, int d, int dt, int out_dt, hipStream_t s);
hipError_t launch_adapt(const AdaptArgs& a, hipStream_t s);

// cc_scan backward outputs from the dense backward's fp32 results: dq, dk, dv
// rounded to bf16 (the primal dtype), dalpha = dg / alpha (g = log alpha),
// dbeta32 = dbeta / 32 on each of the 32 columns (beta = their mean).
struct CcFinishArgs {
  const float* dq32;
  const float* dk32;
  const float* dv32;
  const float* dg;
  const float* dbeta;
  const float* alpha;
  void* dq;                // bf16
  void* dk;
  void* dv;
  float* dalpha;
  float* dbeta32;
  int64_t n;               // T * H * d
  int64_t n_tok_heads;     // T * H
};
hipError_t launch_cc_finish(const CcFinishArgs& a, hipStream_t s);

// Sets the calling thread's error message and returns `code` (kda_last_error).
int api_fail(int code, const char* msg);

// Whether something a call writes shares memory with another of its arguments.
struct Bytes {
  const void* p;
  size_t n;
};
inline bool overlap(std::initializer_list<Bytes> written, std::initializer_list<Bytes> read) {
  auto meet = [](const Bytes& x, const Bytes& y) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x.p), b = reinterpret_cast<uintptr_t>(y.p);
    return x.p && y.p && x.n && y.n && (a < b ? b - a < x.n : a - b < y.n);
  };
  for (const Bytes* x = written.begin(); x != written.end(); ++x) {
    for (const Bytes& y : read)
      if (meet(*x, y)) return true;
    for (const Bytes* y = x + 1; y != written.end(); ++y)
      if (meet(*x, *y)) return true;
  }
  return false;
}

// Latent attention, expanded form.  Strides in elements; the last axis of every
// tensor is contiguous.  o, dout, dq are [B,Tq,H,*] and dkv [B,Tk,H,2 dn],
// dkr [B,Tk,dr] contiguous; lse, D are [B,H,Tq] fp32.  Packed calls (cu_q
// non-null): B == 1 and n_seqs sequences, rows cu[i] .. cu[i+1].
struct LatentArgs {
  const void* q;           // [B,Tq,H,dn+dr]
  const void* kv;          // [B,Tk,H,dn+dn]: nope key | value
  const void* kr;          // [B,Tk,dr]: the rotary key of all heads
  const int32_t* cu_q;
  const int32_t* cu_k;
  int n_seqs;
  int B, Tq, Tk, H;
  int64_t q_b, q_t, q_h, kv_b, kv_t, kv_h, kr_b, kr_t;
  int causal;
  float scale;
  void* o;
  float* lse;
  // Few blocks: up to `splits` workgroups a block, each with a share of the
  // other axis, leave fp32 parts that a join adds (forward: also the maxima
  // and sums); part index z, then [B*H][rows][width].
  int splits, share, live; // share: its tiles, live: the shares of a head; 0: `splits` equal shares of a block
  float* part;
  float* part_ml;
  // backward
  const void* o_in;
  const void* dout;
  const float* lse_in;
  float* D;                // sum over dn of do * o
  float* dkr_part;         // [splits][B,H,Tk,dr]: each head's share of the rotary key's gradient
  int splits_k, share_k, live_k;   // the key pass' (those above and `part` are the query pass')
  float* part_k;
  void* dq;
  void* dkv;
  void* dkr;
};
hipError_t launch_latent_fwd(const LatentArgs& a, int dn, int dr, int dt, hipStream_t s);
hipError_t launch_latent_bwd(const LatentArgs& a, int dn, int dr, int dt, hipStream_t s);

// New rows of the latent cache: RMS norm of the first R elements (w null: none),
// rotation of the last dr, stored at row slots[i] of the cache (outside
// [0, n_slots): not stored); the queries' rotary parts rotated to q_out.
struct LatentAppendArgs {
  const void* rows;        // [N, R+dr], row stride rows_t
  const int64_t* positions;  // [N]
  const int64_t* slots;    // [N]
  const float* cos_sin;    // [P, dr]: cos of the dr/2 angles | sin
  const float* w;          // [R] or null
  void* cache;             // [n_slots, R+dr]
  const void* q;           // [N, H, dr] with strides, or null
  void* q_out;
  int64_t rows_t, q_t, q_h, qo_t, qo_h, n_slots, P;
  int N, H, interleaved;
  float eps;
};
hipError_t launch_latent_append(const LatentAppendArgs& a, int R, int dr, int dt, hipStream_t s);

// Latent attention, absorbed form over the paged cache.
struct LatentDecodeArgs {
  const void* q;           // [B,Tq,H,R+dr]
  const void* cache;       // [n_pages, page, R+dr]
  const int32_t* table;    // [B, per]
  const int32_t* lens;     // [B]
  void* o;                 // [B,Tq,H,R]
  float* lse;              // [B,Tq,H]
  float* part_o;           // partial results of split sequences
  float* part_ml;
  int* line;               // tiles of a run, then each sequence's first tile on the line
  int whole;               // a workgroup a sequence: nothing to join
  int least;               // fewest places of a run
  int pad;                 // places of a sequence beside its tiles
  int B, Tq, H, per, page_shift;
  int64_t n_pages;
  int groups, wgs;         // row groups of a sequence; workgroups along the cache
  float scale;
  // a tree of drafts (N = Tq places): [B, Tq] in tree calls, which the last field is for too
  const int32_t* parents;
  int items;               // 0: wgs a multiple of eight or one group; else the workgroups in use, of a multiple of eight
};
int latent_decode_tile(int m_rows);   // keys of a tile, by the query rows of a workgroup
hipError_t launch_latent_decode(const LatentDecodeArgs& a, int R, int dr, int dt, int m_rows, hipStream_t s);
hipError_t launch_latent_tree_decode(const LatentDecodeArgs& a, int R, int dr, int dt, int m_rows, hipStream_t s);

// The latent cache after an accepted path (include/tree_mi355x.h).
struct LatentTreeCommitArgs {
  char* cache;             // [layers, n_pages, page, row_bytes]
  const int32_t* table;    // [B, per]
  const int32_t* lens;     // [B]
  const int32_t* parents;  // [B, N]
  const int32_t* last;     // [B]
  int32_t* new_lens;       // [B]
  int layers, B, N, per, page_shift, row_bytes;
  int64_t n_pages;
};
hipError_t launch_latent_tree_commit(const LatentTreeCommitArgs& a, hipStream_t s);

// A tree of N places over the state: o, u [B,N,H,d] and the state as it was.
struct TreeStepArgs {
  const void* q;           // [B,N,H,d]
  const void* k;
  const void* v;
  const void* g;
  const void* beta;        // [B,N,H]
  const int32_t* parents;  // [B,N]
  const float* state;      // [B,H,d,d]
  void* o;
  float* u;
  int B, N, H;
  float scale;
};
hipError_t launch_tree_step(const TreeStepArgs& a, int d, int dt, int out_dt, hipStream_t s);

struct TreeCommitArgs {
  const void* k;           // [B,N,H,d]
  const void* g;
  const float* u;
  const int32_t* parents;  // [B,N]
  const int32_t* last;     // [B]
  float* state;            // [B,H,d,d], in place
  int B, N, H;
};
hipError_t launch_tree_commit(const TreeCommitArgs& a, int d, int dt, hipStream_t s);

// Verification: a row is cut into `slices` of `per` entries, a workgroup each.
struct TreeVerifyArgs {
  const void* target;      // [B,N+1,V] with strides
  const void* draft;       // [B,N,V] with strides, or null
  const int64_t* tokens;   // [B,N]
  const int32_t* parents;  // [B,N]
  const float* uniforms;   // [B,N+1]; null: greedy
  int32_t* last;
  int64_t* next;
  int32_t* accepted;
  int64_t t_b, t_row, d_b, d_row;
  int B, N, V, slices, per;
  void* ws;
};
hipError_t launch_tree_verify(const TreeVerifyArgs& a, int dt, hipStream_t s);

}  // namespace kda

// Entry points of the package's own binding (axiom_amd/_lib.py), outside the C
// ABI: kda_chunk_bwd and kda_prologue_bwd with the outputs' types chosen by
// the caller.  dq, dk, dv in qkv_grad_dtype (KDA_DTYPE_F32 or the dtype of q,
// k, v), dg and dbeta in gate_grad_dtype (F32 or the dtype of g, beta); dqp,
// dkp, dvp in dx_dtype (F32 or in_dtype).  A 16-bit gradient is the fp32 one
// rounded to nearest even by the kernel that forms it.  And
// kda_cc_scan_bwd_batched for fresh outputs: where alpha and beta32 are aligned
// to 16 bytes and T > 0 it needs kda_chunk_bwd_workspace's bytes only (the seam's
// own query keeps room for the two-pass form: at B2 T8192 H12 d128 half a GB more).
extern "C" {
__attribute__((visibility("default"))) int axiom_cc_scan_bwd(
    hipStream_t stream, const void* q, const void* k, const void* v, const float* alpha, const float* beta32,
    const float* S_in, const float* d_o, const float* dS, void* dq, void* dk, void* dv, float* dalpha, float* dbeta32,
    float* dS_in, int B, int T, int H, int dk_dim, int dv_dim, int tile, int chunk, void* workspace,
    size_t workspace_bytes);
__attribute__((visibility("default"))) int axiom_chunk_bwd(
    hipStream_t stream, const void* q, const void* k, const void* v, const void* g, const void* beta, const float* h0,
    const void* dout, const float* dht, void* dq, void* dk, void* dv, void* dg, void* dbeta, float* dh0, int B, int T,
    int H, int dk_dim, int dv_dim, int chunk, float scale, int in_dtype, int dout_dtype, int qkv_grad_dtype,
    int gate_grad_dtype, void* workspace, size_t workspace_bytes);
__attribute__((visibility("default"))) int axiom_prologue_bwd(
    hipStream_t stream, const void* qp, const void* kp, const void* vp, const float* wq, const float* wk,
    const float* wv, const float* bq_in, const float* bk_in, const float* bv_in, const float* dq, const float* dk,
    const float* dv, void* dqp, void* dkp, void* dvp, float* dwq, float* dwk, float* dwv, float* dbq, float* dbk,
    float* dbv, int B, int T, int H, int d, int K, int in_dtype, int dx_dtype, void* workspace, size_t workspace_bytes);
}
