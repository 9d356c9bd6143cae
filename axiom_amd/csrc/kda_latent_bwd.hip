// Latent attention, expanded form, backward.
//
//   D_i = sum_d do_id o_id,   p_ij = exp(scale s_ij - lse_i),
//   g_ij = p_ij (do_i . v_j - D_i),
//   dq_i = scale sum_j g_ij k_j,  dk_j = scale sum_i g_ij q_i,  dv_j = sum_i p_ij do_i,
// the rotary key's gradient summed over the heads.
//
// Three launches, no atomics, so a gradient is the same bits in every run: the
// query pass (a workgroup owns 128 queries and walks the keys; D, dq), the key
// pass (a workgroup owns 128 keys and walks the queries; dk, dv, the head's share
// of the rotary key's gradient in fp32), then the sums in fixed order: that
// share's over the heads, and the parts of blocks that were shared out.  Both
// passes form p and g again: seven products instead of five, against an fp32 dq
// kept in memory and added to by every key block.
//
// p and g are rounded to the inputs' type for the products they enter; sums
// are fp32.  fp16, whose values lie between 6e-8 and 65504, takes g times a power
// of two of its own for every column of g, that is for every query in the query
// pass and every key in the key pass: as a running maximum, it follows the
// column's largest |g| so far, and the column's sum is rescaled where it falls.
// What a query's do or another sequence holds is then nothing to a key that does
// not see it, and neither a small do nor large values cost the operand its range.

#include "kda_internal.h"
#include "kda_latent.h"

namespace kda {
namespace latent {

// fp16: a column's factor.  It starts high, and where the largest |g| times it
// passes 2^15 it becomes the power of two that brings that |g| into [2^10, 2^11),
// five powers below, so that it seldom changes.  A |g| that is not finite leaves it.
constexpr float kFactor0 = 0x1p100f;
__device__ __forceinline__ bool past(float top, float f) { return top * f > 0x1p15f; }
__device__ __forceinline__ float factor(float top, float f) {
  return past(top, f) && top <= 3.4028234e38f ? __uint_as_float((264u << 23) - (__float_as_uint(top) & 0x7F800000u)) : f;
}
__device__ __forceinline__ float inverse(float f) { return __uint_as_float((254u << 23) - __float_as_uint(f)); }   // of a power of two

template <int DT, int DN, int DR>
struct BwdCfg {
  static constexpr int ES = El<DT>::ES;
  static constexpr int NW = 4, BM = 32 * NW;     // rows that a workgroup owns
  static constexpr int BN = ES == 2 ? 64 : 32;   // rows of the other side at a time
  typedef Tile<DN, ES> TN;
  typedef Tile<DR, ES> TR;
  static constexpr int OFF_V = TN::bytes(BN), OFF_R = 2 * TN::bytes(BN);
  static constexpr int OFF_L = OFF_R + TR::bytes(BN);          // key pass: lse, then D, 64 floats each
  static constexpr int BUF_Q = OFF_L, BUF_K = OFF_L + 512;
};

// -------------------------------------------------------------- query pass
// As the forward: scores transposed, one query a lane column.  g^T is the second
// operand of dq^T += K^T g^T, whose first operand is the key tile read transposed.
// Bound by the products and the waits between them: B4 H16 T4096, d 128 + 64, bf16,
// causal 604 us, 910 TFLOP/s of its three products.  s and do v^T of 32 keys at a time:
// with queries, do and the sums in registers (256 in all) 64 would spill.
template <int DT, int DN, int DR>
__global__ __launch_bounds__(256, El<DT>::ES == 2 ? 2 : 1) void kda_latent_dq_kernel(LatentArgs a, int nqb) {
  typedef BwdCfg<DT, DN, DR> C;
  typedef typename El<DT>::frag F;
  typedef typename El<DT>::t E;
  constexpr int ES = C::ES, BN = C::BN, KN = DN / 16, KR = DR / 16, ND = DN / 32, NR = DR / 32;
  __shared__ __attribute__((aligned(1024))) char buf0[C::BUF_Q];
  __shared__ __attribute__((aligned(1024))) char buf1[C::BUF_Q];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 31, h = lane >> 5;
  Where w;
  int z;
  if (!locate_share(a, nqb, C::BM, BN, true, true, w, z)) return;
  const int nk = w.ke - w.k0;
  const int row = w.r0 + wave * 32 + m;
  const bool live = row < w.re;
  const int crow = min(row, w.re - 1);
  const int kmax = a.causal ? min(nk - 1, row + w.off) : nk - 1;
  const int wave_lo = a.causal ? min(nk - 1, w.r0 + wave * 32 + w.off) : nk - 1;
  const int wave_hi = a.causal ? min(nk - 1, min(w.r0 + wave * 32 + 31, w.re - 1) + w.off) : nk - 1;
  const int blk_hi = a.causal ? min(nk - 1, min(w.r0 + C::BM - 1, w.re - 1) + w.off) : nk - 1;
  const Share part(max(0, (blk_hi + BN) / BN), a.splits, a.share, z);
  const int nt = part.j1;
  if (z >= part.parts) return;   // never share 0, which also leaves D

  F qn[KN], qr[KR], dO[KN];
  {
    const E* qp = static_cast<const E*>(a.q) + w.b * a.q_b + static_cast<int64_t>(crow) * a.q_t + w.head * a.q_h;
    const E* dp = static_cast<const E*>(a.dout) + ((static_cast<int64_t>(w.b) * a.Tq + crow) * a.H + w.head) * DN;
#pragma unroll
    for (int s = 0; s < KN; ++s) {
      qn[s] = *reinterpret_cast<const F*>(qp + 16 * s + 8 * h);
      dO[s] = *reinterpret_cast<const F*>(dp + 16 * s + 8 * h);
    }
#pragma unroll
    for (int s = 0; s < KR; ++s) qr[s] = *reinterpret_cast<const F*>(qp + DN + 16 * s + 8 * h);
  }
  const int64_t ri = static_cast<int64_t>(w.bh) * a.Tq + crow;
  const float lse2 = a.lse_in[ri] * kLog2e;
  float D = 0.f, gf = kFactor0;   // D of this lane's query, for the key pass too, and the factor of its g
  {
    const E* op = static_cast<const E*>(a.o_in) + ((static_cast<int64_t>(w.b) * a.Tq + crow) * a.H + w.head) * DN;
#pragma unroll
    for (int s = 0; s < KN; ++s) {
      const F o = *reinterpret_cast<const F*>(op + 16 * s + 8 * h);
#pragma unroll
      for (int e = 0; e < 8; ++e) D = fmaf(static_cast<float>(dO[s][e]), static_cast<float>(o[e]), D);
    }
    D = half_sum(D);
  }

  const char* kvp = static_cast<const char*>(a.kv) + (w.b * a.kv_b + w.k0 * a.kv_t + w.head * a.kv_h) * ES;
  const char* krp = static_cast<const char*>(a.kr) + (w.b * a.kr_b + w.k0 * a.kr_t) * ES;
  const unsigned kv_rb = static_cast<unsigned>(a.kv_t * ES), kr_rb = static_cast<unsigned>(a.kr_t * ES);
  Copy<typename C::TN, BN, C::NW> cn;
  Copy<typename C::TR, BN, C::NW> cr;
  cn.init(wave, lane, kv_rb);
  cr.init(wave, lane, kr_rb);
  auto fetch = [&](int j, char* dst) {
    const char* s = kvp + static_cast<int64_t>(j) * BN * kv_rb;
    const char* r = krp + static_cast<int64_t>(j) * BN * kr_rb;
    if (j * BN + BN <= nk) {
      cn.issue(s, dst, wave, kv_rb);
      cn.issue(s + DN * ES, dst + C::OFF_V, wave, kv_rb);
      cr.issue(r, dst + C::OFF_R, wave, kr_rb);
    } else {
      const int last = nk - 1 - j * BN;
      cn.issue_last(s, dst, wave, lane, kv_rb, last);
      cn.issue_last(s + DN * ES, dst + C::OFF_V, wave, lane, kv_rb, last);
      cr.issue_last(r, dst + C::OFF_R, wave, lane, kr_rb, last);
    }
  };

  const float c = a.scale * kLog2e;
  // Rows of few keys: D as sum_j p_j (do . v_j), not from the rounded o, whose
  // error is as large as g's own rounding there and falls with the keys' number.
  // dq's error over that of its result's rounding, d 64, causal, where g's rounding
  // alone makes it sqrt 2: rows 0 to 31 1.47 with this and 1.87 (fp16 1.43 and 1.75)
  // with o's D, 32 to 63 1.44 and 1.57, 64 to 127 1.43 and 1.52; 128 to 255 1.48 with o's.
  // So it ends there, with two tiles, both in LDS.  It costs 8 us of 150 where every
  // row is such a one (B64 H16 T128) and nothing measurable at T = 1000.
  if (ES == 2 && blk_hi < 2 * BN && nt > 0) {   // a walk this short is never shared out
    fetch(0, buf0);
    if (nt == 2) fetch(1, buf1);
    wait_vmem_all();
    lds_barrier();
    float d = 0.f;
    for (int x = 0; x < BN * nt; x += 32) {
      const char* cur = x < BN ? buf0 : buf1;
      const int r0 = x & (BN - 1), ln = fresh(lane), fm = ln & 31, fh = ln >> 5;
      f16v s, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = dp[i] = 0.f;
#pragma unroll
      for (int k = 0; k < KN; ++k) {
        s = mma(s, C::TN::template row_frag<F>(cur, fm, k, fh, r0), qn[k]);
        dp = mma(dp, C::TN::template row_frag<F>(cur + C::OFF_V, fm, k, fh, r0), dO[k]);
      }
#pragma unroll
      for (int k = 0; k < KR; ++k) s = mma(s, C::TR::template row_frag<F>(cur + C::OFF_R, fm, k, fh, r0), qr[k]);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        d += x + 8 * (i >> 2) + 4 * h + (i & 3) <= kmax ? fast_exp2(fmaf(s[i], c, -lse2)) * dp[i] : 0.f;
    }
    D = half_sum(d);
    lds_barrier();
  }
  if (z == 0 && live && h == 0) a.D[ri] = D;
  f16v acc[ND + NR];
#pragma unroll
  for (int n = 0; n < ND + NR; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[n][i] = 0.f;

  auto step = [&](int j, const char* cur, char* nxt) {
    wait_vmem_all();
    lds_barrier();
    if (j + 1 < nt) fetch(j + 1, nxt);
    const int kt = j * BN;
    if (kt > wave_hi) return;
    const int ln = fresh(lane), fm = ln & 31, fh = ln >> 5;
#pragma unroll
    for (int t = 0; t < BN / 32; ++t) {
      f16v s, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = dp[i] = 0.f;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < KN; ++k) {
        s = mma(s, C::TN::template row_frag<F>(cur, fm, k, fh, 32 * t), qn[k]);
        dp = mma(dp, C::TN::template row_frag<F>(cur + C::OFF_V, fm, k, fh, 32 * t), dO[k]);
      }
#pragma unroll
      for (int k = 0; k < KR; ++k) s = mma(s, C::TR::template row_frag<F>(cur + C::OFF_R, fm, k, fh, 32 * t), qr[k]);
      if constexpr (ES == 2) pace<2 * KN + KR, 4, 1, 1>();
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = fast_exp2(fmaf(s[i], c, -lse2)) * (dp[i] - D);
      if (kt + 32 * t + 31 > wave_lo) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (kt + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3) > kmax) s[i] = 0.f;
      }
      if constexpr (DT == 2) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(s[i]));
        top = half_max(top);
        if (__any(past(top, gf))) {
          const float nf = factor(top, gf), al = nf * inverse(gf);
          gf = nf;
#pragma unroll
          for (int n = 0; n < ND + NR; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[n][i] *= al;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] *= gf;
      }
      F gq[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float g[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = s[8 * u + e];
        gq[u] = to_frag<DT>(g);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int n = 0; n < ND; ++n)
          acc[n] = mma(acc[n], C::TN::template col_frag<F>(cur, 32 * t + 16 * u, 32 * n, ln), gq[u]);
#pragma unroll
        for (int n = 0; n < NR; ++n)
          acc[ND + n] = mma(acc[ND + n], C::TR::template col_frag<F>(cur + C::OFF_R, 32 * t + 16 * u, 32 * n, ln), gq[u]);
      }
      if constexpr (ES == 2) pace<2 * (ND + NR), 3, 2, 1>();
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (part.j0 < nt) fetch(part.j0, buf0);
  for (int j = part.j0; j < nt;) {
    step(j, buf0, buf1);
    if (++j >= nt) break;
    step(j, buf1, buf0);
    ++j;
  }
  if (!live) return;
  if (kmax < part.j0 * BN) {   // no visible key: zeros, whatever 0 times the others' values made
#pragma unroll
    for (int n = 0; n < ND + NR; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[n][i] = 0.f;
  }
  const float f = DT == 2 ? a.scale * inverse(gf) : a.scale;
  if (part.parts > 1) {
    const int64_t pb = ((static_cast<int64_t>(z) * a.B * a.H + w.bh) * a.Tq + row) * (DN + DR) + 4 * h;
#pragma unroll
    for (int n = 0; n < ND + NR; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        store4<0>(a.part, pb + 32 * n + 8 * i, acc[n][4 * i] * f, acc[n][4 * i + 1] * f, acc[n][4 * i + 2] * f,
                  acc[n][4 * i + 3] * f);
    return;
  }
  const int64_t ob = ((static_cast<int64_t>(w.b) * a.Tq + row) * a.H + w.head) * (DN + DR) + 4 * h;
#pragma unroll
  for (int n = 0; n < ND + NR; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      store4<DT>(a.dq, ob + 32 * n + 8 * i, acc[n][4 * i] * f, acc[n][4 * i + 1] * f, acc[n][4 * i + 2] * f,
                 acc[n][4 * i + 3] * f);
}

// ---------------------------------------------------------------- key pass
// Scores untransposed: a lane column is one key; the query tile (nope, rotary,
// do) is in LDS, read by rows for the two score products and transposed for
// dk^T and dv^T.  Bound as the query pass: B4 H16 T4096, d 128 + 64, bf16, causal
// 838 us, 820 TFLOP/s of its four products (804 at the least).
//
// 16-bit types: a pair of waves owns 32 keys and splits the work by what it
// holds.  The first wave holds the keys and dv (112 registers): s, p, dv += p
// do.  The second holds the values and dk (128): do v^T, and, a tile behind, with
// p from the first, g and dk += g q.  Each has half of the products, the two
// share a SIMD, and one wave's exponentials run under the other's products; a
// wave that holds all of it (240 registers and the scores) is alone on its SIMD
// and had the matrix cores busy 32 % of the time.  A tile behind, because with p
// handed over inside a tile's turn both waves wait twice for each other (40 %).
// p carries a factor of 2^12 (dv and g take it out).  bf16: it crosses in fp16,
// within 2^-11 of itself down to 2^-26, an eighth of the rounding that g gets
// next.  fp16: it crosses in fp32, since another rounding of g's own size made
// dk's error 1.2 times what it has to be.  Its two tiles by parity do not fit
// beside d = 128's buffers: there one place serves both, and a second barrier in
// the middle of a turn parts the second wave's reads, before its dk products,
// from the first wave's writes, after its exponentials (both passes, fp16: B4 H16
// T4096 1468 us with p in fp16 and 1513 with this; 24 packed sequences of 17 to
// 1024 tokens, H8, 135 and 143).
// Three query tiles in LDS: arriving, present, behind.  A pair takes every tile of
// its block's walk, also the one at the diagonal that none of its keys are seen by.
// fp32: operands twice as large and products 16 times as slow, so one wave does it all.
template <int DT, int DN, int DR>
struct KeyCfg : BwdCfg<DT, DN, DR> {
  typedef BwdCfg<DT, DN, DR> B;
  static constexpr bool PAIR = B::ES == 2;
  static constexpr int NT = PAIR ? 512 : 256, NWV = NT / 64;
  static constexpr int P_LOG2 = PAIR ? 12 : 0;            // p's factor
  static constexpr int P_ES = DT == 2 ? 4 : 2, P_PAIR = 64 * 32 * P_ES;   // p of a tile, a pair's: in fp32 or fp16
  static constexpr int P_BUFS = DT == 2 && DN == 128 ? 1 : 2;             // by tile parity, or one place and a barrier more
  static constexpr int P_BYTES = PAIR ? 4 * P_PAIR : 16;
};

template <int DT, int DN, int DR>
__global__ __launch_bounds__((KeyCfg<DT, DN, DR>::NT)) void kda_latent_dkv_kernel(LatentArgs a, int nkb) {
  typedef KeyCfg<DT, DN, DR> C;
  typedef typename El<DT>::frag F;
  typedef typename El<DT>::t E;
  constexpr int ES = C::ES, BN = C::BN, KN = DN / 16, KR = DR / 16, ND = DN / 32, NR = DR / 32, NWV = C::NWV, NTL = BN / 32;
  __shared__ __attribute__((aligned(1024))) char buf0[C::BUF_K];
  __shared__ __attribute__((aligned(1024))) char buf1[C::BUF_K];
  __shared__ __attribute__((aligned(1024))) char buf2[C::PAIR ? C::BUF_K : 16];
  __shared__ __attribute__((aligned(1024))) char pbuf[C::P_BUFS][C::P_BYTES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 31, h = lane >> 5, own = wave & 3, role = wave >> 2;
  Where w;
  int z;
  if (!locate_share(a, nkb, C::BM, BN, false, false, w, z)) return;
  const int nq = w.ke - w.k0;                   // queries of the sequence
  const int key = w.r0 + own * 32 + m;          // this lane's key (packed axis)
  const bool live = key < w.re;
  const int ckey = min(key, w.re - 1);
  const int first = a.causal ? max(0, key + w.off) : 0;                     // first query that sees this lane's key
  const int wave_first = a.causal ? max(0, w.r0 + own * 32 + w.off) : 0;    // ... any of the wave's keys
  const int wave_full = a.causal ? max(0, min(w.r0 + own * 32 + 31, w.re - 1) + w.off) : 0;   // ... all of them
  const int jf = (a.causal ? max(0, w.r0 + w.off) : 0) / BN;                // the block's first query tile
  const Share part(max(0, (nq + BN - 1) / BN - jf), a.splits_k, a.share_k, z);
  if (z >= part.parts) return;
  const int j0 = jf + part.j0, nt = jf + part.j1;
  const float c = a.scale * kLog2e;
  constexpr float unp = 1.f / (1 << C::P_LOG2);

  const char* qp = static_cast<const char*>(a.q) + (w.b * a.q_b + w.k0 * a.q_t + w.head * a.q_h) * ES;
  const char* dp_ = static_cast<const char*>(a.dout) + ((static_cast<int64_t>(w.b) * a.Tq + w.k0) * a.H + w.head) * DN * ES;
  const float* lsep = a.lse_in + static_cast<int64_t>(w.bh) * a.Tq + w.k0;
  const float* Dp = a.D + static_cast<int64_t>(w.bh) * a.Tq + w.k0;
  const unsigned q_rb = static_cast<unsigned>(a.q_t * ES), d_rb = static_cast<unsigned>(a.H * DN * ES);
  Copy<typename C::TN, BN, NWV> cq, cd;
  Copy<typename C::TR, BN, NWV> cr;
  cq.init(wave, lane, q_rb);
  cd.init(wave, lane, d_rb);
  cr.init(wave, lane, q_rb);
  auto fetch = [&](int j, char* dst) {
    const char* s = qp + static_cast<int64_t>(j) * BN * q_rb;
    const char* d = dp_ + static_cast<int64_t>(j) * BN * d_rb;
    if (j * BN + BN <= nq) {
      cq.issue(s, dst, wave, q_rb);
      cd.issue(d, dst + C::OFF_V, wave, d_rb);
      cr.issue(s + DN * ES, dst + C::OFF_R, wave, q_rb);
    } else {
      const int last = nq - 1 - j * BN;
      cq.issue_last(s, dst, wave, lane, q_rb, last);
      cd.issue_last(d, dst + C::OFF_V, wave, lane, d_rb, last);
      cr.issue_last(s + DN * ES, dst + C::OFF_R, wave, lane, q_rb, last);
    }
    if (wave < 2) {
      const float* x = wave == 0 ? lsep : Dp;
      copy4(x + min(j * BN + lane, nq - 1), dst + C::OFF_L + 256 * wave);
    }
  };
  // a tile's turn: its copies are there, the next ones are on their way
  auto turn = [&](int j, char* nxt) {
    wait_vmem_all();
    lds_barrier();
    if (j + 1 < nt) fetch(j + 1, nxt);
  };

  const E* kp = static_cast<const E*>(a.kv) + w.b * a.kv_b + static_cast<int64_t>(ckey) * a.kv_t + w.head * a.kv_h + 8 * h;
  const E* rp = static_cast<const E*>(a.kr) + w.b * a.kr_b + static_cast<int64_t>(ckey) * a.kr_t + 8 * h;
  const int64_t ob = ((static_cast<int64_t>(w.b) * a.Tk + key) * a.H + w.head) * (2 * DN) + 4 * h;
  float gf = kFactor0;                                    // fp16: factor of this lane's key, above p's

  // p of a score tile, from s; rows q0 .. of the sequence, rows 32 t .. of the tile
  auto probs = [&](const char* cur, int q0, int t, int fh, bool edge, f16v& s) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const f4 ls = *reinterpret_cast<const f4*>(cur + C::OFF_L + (32 * t + 8 * v + 4 * fh) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[4 * v + e] = fast_exp2(fmaf(s[4 * v + e], c, fmaf(-ls[e], kLog2e, C::P_LOG2)));
    }
    if (edge) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int qi = q0 + 8 * (i >> 2) + 4 * h + (i & 3);
        if (qi < first || qi >= nq) s[i] = 0.f;
      }
    }
  };
  // g from p and do v^T (0 where p is: a masked pair's do v^T need not be finite)
  auto adjoint = [&](const char* cur, int t, int fh, bool edge, const f16v& p, f16v& dp) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const f4 dd = *reinterpret_cast<const f4*>(cur + C::OFF_L + 256 + (32 * t + 8 * v + 4 * fh) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * v + e;
        const float g = p[i] * (dp[i] - dd[e]);
        dp[i] = edge && p[i] == 0.f ? 0.f : g;
      }
    }
  };
  auto frags = [&](const f16v& x, F (&out)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = x[8 * u + e];
      out[u] = to_frag<DT>(y);
    }
  };
  auto zero = [](f16v& x) {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 0.f;
  };
  // dv, dk and the rotary part of this lane's key, or this share's parts of them
  const bool parted = part.parts > 1;
  const int64_t prow = (static_cast<int64_t>(z) * a.B * a.H + w.bh) * a.Tk + key;
  auto put4 = [&](int col, float x, float y, float z, float u) {
    if (parted) store4<0>(a.part_k, prow * (2 * DN) + 4 * h + col, x, y, z, u);
    else store4<DT>(a.dkv, ob + col, x, y, z, u);
  };
  auto put_dv = [&](const f16v (&dv)[ND]) {
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) put4(DN + 32 * n + 8 * i, dv[n][4 * i] * unp, dv[n][4 * i + 1] * unp, dv[n][4 * i + 2] * unp, dv[n][4 * i + 3] * unp);
  };
  auto put_dk = [&](const f16v (&dk)[ND + NR]) {
    const float f = DT == 2 ? a.scale * unp * inverse(gf) : a.scale * unp;
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        put4(32 * n + 8 * i, dk[n][4 * i] * f, dk[n][4 * i + 1] * f, dk[n][4 * i + 2] * f, dk[n][4 * i + 3] * f);
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        store4<0>(a.dkr_part, prow * DR + 4 * h + 32 * n + 8 * i, dk[ND + n][4 * i] * f, dk[ND + n][4 * i + 1] * f,
                  dk[ND + n][4 * i + 2] * f, dk[ND + n][4 * i + 3] * f);
  };

  if (j0 < nt) fetch(j0, buf0);
  if constexpr (C::PAIR) {
    const int mine = own * C::P_PAIR + lane * 16;
    constexpr bool MID = C::P_BUFS == 1;
    auto place_of = [&](int j) -> char* { return pbuf[MID ? 0 : j & 1] + mine; };
    if (role == 0) {
      F kn[KN], kr[KR];
#pragma unroll
      for (int s = 0; s < KN; ++s) kn[s] = *reinterpret_cast<const F*>(kp + 16 * s);
#pragma unroll
      for (int s = 0; s < KR; ++s) kr[s] = *reinterpret_cast<const F*>(rp + 16 * s);
      f16v dv[ND];
#pragma unroll
      for (int n = 0; n < ND; ++n) zero(dv[n]);
      auto step = [&](int j, const char* cur, char* nxt) {
        turn(j, nxt);
        const int qt = j * BN;
        const int ln = fresh(lane), fm = ln & 31, fh = ln >> 5;
        if (j < nt) {
          F pf[2][2];
          f16v s[2];
          zero(s[0]);
          zero(s[1]);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int k = 0; k < KN; ++k)
#pragma unroll
            for (int t = 0; t < 2; ++t) s[t] = mma(s[t], C::TN::template row_frag<F>(cur, fm, k, fh, 32 * t), kn[k]);
#pragma unroll
          for (int k = 0; k < KR; ++k)
#pragma unroll
            for (int t = 0; t < 2; ++t) s[t] = mma(s[t], C::TR::template row_frag<F>(cur + C::OFF_R, fm, k, fh, 32 * t), kr[k]);
          pace<2 * (KN + KR), 6, 1, 1>();
          __builtin_amdgcn_sched_barrier(0);
          const bool edge = qt < wave_full || qt + BN > nq;
          auto hand_over = [&](int t) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              char* const to = place_of(j) + (2 * t + u) * (512 * C::P_ES);
              if constexpr (DT == 2) {
#pragma unroll
                for (int v = 0; v < 2; ++v)
                  *reinterpret_cast<f4*>(to + 1024 * v) = f4{s[t][8 * u + 4 * v], s[t][8 * u + 4 * v + 1], s[t][8 * u + 4 * v + 2], s[t][8 * u + 4 * v + 3]};
              } else {
                h8 x;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = static_cast<_Float16>(s[t][8 * u + e]);
                *reinterpret_cast<h8*>(to) = x;
              }
            }
          };
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (edge) probs(cur, qt + 32 * t, t, fh, true, s[t]);
            else probs(cur, qt + 32 * t, t, fh, false, s[t]);
            frags(s[t], pf[t]);
            if constexpr (!MID) hand_over(t);
          }
          if constexpr (MID) {
            __builtin_amdgcn_sched_barrier(0);
            reuse_barrier();                      // the second wave has read the last tile's p
            hand_over(0);
            hand_over(1);
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int n = 0; n < ND; ++n)
              dv[n] = mma(dv[n], C::TN::template col_frag<F>(cur + C::OFF_V, 16 * u, 32 * n, ln), pf[u >> 1][u & 1]);
          pace<4 * ND, 4, 2, 1>();
          __builtin_amdgcn_sched_barrier(0);
        } else if constexpr (MID) {
          reuse_barrier();
        }
      };
      for (int j = j0; j < nt + 1 && j0 < nt;) {
        step(j, buf0, buf1);
        if (++j > nt) break;
        step(j, buf1, buf2);
        if (++j > nt) break;
        step(j, buf2, buf0);
        ++j;
      }
      if (live) put_dv(dv);
    } else {
      F vv[KN];
#pragma unroll
      for (int s = 0; s < KN; ++s) vv[s] = *reinterpret_cast<const F*>(kp + DN + 16 * s);
      f16v dk[ND + NR];
#pragma unroll
      for (int n = 0; n < ND + NR; ++n) zero(dk[n]);
      f16v dp[2];
      auto step = [&](int j, const char* cur, const char* prev, char* nxt) {
        turn(j, nxt);
        const int ln = fresh(lane), fm = ln & 31, fh = ln >> 5;
        const int qp = (j - 1) * BN;
        if (j > j0) {
          F gq[2][2];
          const bool edge = qp < wave_full || qp + BN > nq;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            f16v p;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const char* const from = place_of(j - 1) + (2 * t + u) * (512 * C::P_ES);
              if constexpr (DT == 2) {
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                  const f4 x = *reinterpret_cast<const f4*>(from + 1024 * v);
#pragma unroll
                  for (int e = 0; e < 4; ++e) p[8 * u + 4 * v + e] = x[e];
                }
              } else {
                const h8 x = *reinterpret_cast<const h8*>(from);
#pragma unroll
                for (int e = 0; e < 8; ++e) p[8 * u + e] = static_cast<float>(x[e]);
              }
            }
            if (edge) adjoint(prev, t, fh, true, p, dp[t]);
            else adjoint(prev, t, fh, false, p, dp[t]);
            if constexpr (DT != 2) frags(dp[t], gq[t]);
          }
          if constexpr (DT == 2) {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) top = fmaxf(top, fabsf(dp[i >> 4][i & 15]));
            top = half_max(top);
            if (__any(past(top, gf))) {
              const float nf = factor(top, gf), al = nf * inverse(gf);
              gf = nf;
#pragma unroll
              for (int n = 0; n < ND + NR; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) dk[n][i] *= al;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
              for (int i = 0; i < 16; ++i) dp[t][i] *= gf;
              frags(dp[t], gq[t]);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
#pragma unroll
            for (int n = 0; n < ND; ++n)
              dk[n] = mma(dk[n], C::TN::template col_frag<F>(prev, 16 * u, 32 * n, ln), gq[u >> 1][u & 1]);
#pragma unroll
            for (int n = 0; n < NR; ++n)
              dk[ND + n] = mma(dk[ND + n], C::TR::template col_frag<F>(prev + C::OFF_R, 16 * u, 32 * n, ln), gq[u >> 1][u & 1]);
          }
          pace<4 * (ND + NR), 4, 2, 1>();
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (MID) reuse_barrier();     // the last tile's p has been read
        if (j < nt) {
          zero(dp[0]);
          zero(dp[1]);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int k = 0; k < KN; ++k)
#pragma unroll
            for (int t = 0; t < 2; ++t) dp[t] = mma(dp[t], C::TN::template row_frag<F>(cur + C::OFF_V, fm, k, fh, 32 * t), vv[k]);
          pace<2 * KN, 6, 1, 1>();
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      for (int j = j0; j < nt + 1 && j0 < nt;) {
        step(j, buf0, buf2, buf1);
        if (++j > nt) break;
        step(j, buf1, buf0, buf2);
        if (++j > nt) break;
        step(j, buf2, buf1, buf0);
        ++j;
      }
      if (live) put_dk(dk);
    }
  } else {
    F kn[KN], kr[KR], vv[KN];
#pragma unroll
    for (int s = 0; s < KN; ++s) {
      kn[s] = *reinterpret_cast<const F*>(kp + 16 * s);
      vv[s] = *reinterpret_cast<const F*>(kp + DN + 16 * s);
    }
#pragma unroll
    for (int s = 0; s < KR; ++s) kr[s] = *reinterpret_cast<const F*>(rp + 16 * s);
    f16v dk[ND + NR], dv[ND];
#pragma unroll
    for (int n = 0; n < ND + NR; ++n) zero(dk[n]);
#pragma unroll
    for (int n = 0; n < ND; ++n) zero(dv[n]);
    auto step = [&](int j, const char* cur, char* nxt) {
      turn(j, nxt);
      const int qt = j * BN;
      if (qt + BN <= wave_first) return;        // none of these queries sees a key of this wave
      const int ln = fresh(lane), fm = ln & 31, fh = ln >> 5;
      f16v s, dp;
      zero(s);
      zero(dp);
#pragma unroll
      for (int k = 0; k < KN; ++k) {
        s = mma(s, C::TN::template row_frag<F>(cur, fm, k, fh), kn[k]);
        dp = mma(dp, C::TN::template row_frag<F>(cur + C::OFF_V, fm, k, fh), vv[k]);
      }
#pragma unroll
      for (int k = 0; k < KR; ++k) s = mma(s, C::TR::template row_frag<F>(cur + C::OFF_R, fm, k, fh), kr[k]);
      const bool edge = qt < wave_full || qt + BN > nq;
      probs(cur, qt, 0, fh, edge, s);
      adjoint(cur, 0, fh, edge, s, dp);
      F pf[2], gq[2];
      frags(s, pf);
      frags(dp, gq);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          dv[n] = mma(dv[n], C::TN::template col_frag<F>(cur + C::OFF_V, 16 * u, 32 * n, ln), pf[u]);
          dk[n] = mma(dk[n], C::TN::template col_frag<F>(cur, 16 * u, 32 * n, ln), gq[u]);
        }
#pragma unroll
        for (int n = 0; n < NR; ++n)
          dk[ND + n] = mma(dk[ND + n], C::TR::template col_frag<F>(cur + C::OFF_R, 16 * u, 32 * n, ln), gq[u]);
      }
    };
    for (int j = j0; j < nt;) {
      step(j, buf0, buf1);
      if (++j >= nt) break;
      step(j, buf1, buf0);
      ++j;
    }
    if (live) {
      put_dv(dv);
      put_dk(dk);
    }
  }
}

// ------------------------------------------------------------------- sums
// A quarter of a block of one head a workgroup, key blocks first, then (when the
// query pass was shared out) query blocks: the parts of blocks that were shared
// out, in part order, and the rotary key's gradient over the heads and parts,
// whose rows the workgroups of a block's heads divide among themselves.  Bound by
// bytes where there are many: B4 H16 T4096 67 MB of rotary shares in 16 us.
template <int DT, int DN, int DR>
__global__ __launch_bounds__(256) void kda_latent_sums_kernel(LatentArgs a, int nkb, int nqb) {
  typedef BwdCfg<DT, DN, DR> C;
  const int keys = nkb * a.B * a.H;
  const bool q_side = static_cast<int>(blockIdx.x) >= keys;
  Where w;
  if (!locate(a, q_side ? blockIdx.x - keys : blockIdx.x, q_side ? nqb : nkb, C::BM, q_side, false, w)) return;
  const int n_o = w.ke - w.k0;
  int tiles;
  if (q_side) {
    const int hi = a.causal ? min(n_o - 1, min(w.r0 + C::BM - 1, w.re - 1) + w.off) : n_o - 1;
    tiles = max(0, (hi + C::BN) / C::BN);
  } else {
    tiles = max(0, (n_o + C::BN - 1) / C::BN - (a.causal ? max(0, w.r0 + w.off) : 0) / C::BN);
  }
  const int parts = Share(tiles, q_side ? a.splits : a.splits_k, q_side ? a.share : a.share_k, 0).parts;
  const int T = q_side ? a.Tq : a.Tk, ra = w.r0 + blockIdx.y * 32, n = min(32, w.re - ra), WID4 = (q_side ? DN + DR : 2 * DN) / 4;
  const int64_t step = static_cast<int64_t>(a.B) * a.H * T, row0 = static_cast<int64_t>(w.bh) * T + ra;
  if (parts > 1) {
    const float* src = q_side ? a.part : a.part_k;
#pragma unroll 2
    for (int i = threadIdx.x; i < n * WID4; i += 256) {
      const int r = i / WID4, col = i % WID4 * 4;
      f4 s = {0, 0, 0, 0};
#pragma unroll 4
      for (int z = 0; z < parts; ++z) s += *reinterpret_cast<const f4*>(src + (z * step + row0 + r) * (WID4 * 4) + col);
      store4<DT>(q_side ? a.dq : a.dkv, ((static_cast<int64_t>(w.b) * T + ra + r) * a.H + w.head) * (WID4 * 4) + col, s[0], s[1],
                 s[2], s[3]);
    }
  }
  if (q_side) return;
  // rows ra + head, ra + head + H, ..
  const int mine = n > w.head ? (n - w.head + a.H - 1) / a.H : 0;
  for (int i = threadIdx.x; i < mine * (DR / 4); i += 256) {
    const int row = ra + w.head + i / (DR / 4) * a.H, col = i % (DR / 4) * 4;
    const float* p = a.dkr_part + (static_cast<int64_t>(w.b) * a.H * T + row) * DR + col;
    f4 s = {0, 0, 0, 0};
    for (int z = 0; z < parts; ++z)
#pragma unroll 8
      for (int hd = 0; hd < a.H; ++hd) s += *reinterpret_cast<const f4*>(p + (z * step + static_cast<int64_t>(hd) * T) * DR);
    store4<DT>(a.dkr, (static_cast<int64_t>(w.b) * T + row) * DR + col, s[0], s[1], s[2], s[3]);
  }
}

template <int DT, int DN, int DR>
hipError_t run_bwd(const LatentArgs& a, hipStream_t s) {
  constexpr int BM = BwdCfg<DT, DN, DR>::BM;
  const int64_t bh = static_cast<int64_t>(a.B) * a.H;
  const int64_t nqb = a.cu_q ? static_cast<int64_t>(a.Tq) / BM + a.n_seqs : (static_cast<int64_t>(a.Tq) + BM - 1) / BM;
  const int64_t nkb = a.cu_q ? static_cast<int64_t>(a.Tk) / BM + a.n_seqs : (static_cast<int64_t>(a.Tk) + BM - 1) / BM;
  if (bh <= 0) return hipSuccess;
  if (a.Tq > 0)
    kda_latent_dq_kernel<DT, DN, DR><<<a.share > 0 ? dim3(static_cast<unsigned>(a.live * bh)) : dim3(static_cast<unsigned>(nqb * bh), a.splits), dim3(256), 0, s>>>(a, static_cast<int>(nqb));
  if (a.Tk > 0)
    kda_latent_dkv_kernel<DT, DN, DR>
        <<<a.share_k > 0 ? dim3(static_cast<unsigned>(a.live_k * bh)) : dim3(static_cast<unsigned>(nkb * bh), a.splits_k), dim3(KeyCfg<DT, DN, DR>::NT), 0, s>>>(a, static_cast<int>(nkb));
  const int64_t blocks = (nkb + (a.splits > 1 ? nqb : 0)) * bh;
  if (blocks > 0)
    kda_latent_sums_kernel<DT, DN, DR>
        <<<dim3(static_cast<unsigned>(blocks), 4), dim3(256), 0, s>>>(a, static_cast<int>(nkb), static_cast<int>(nqb));
  return hipGetLastError();
}

template <int DT>
hipError_t bwd_by_dims(const LatentArgs& a, int dn, int dr, hipStream_t s) {
  if (dn == 128) return dr == 64 ? run_bwd<DT, 128, 64>(a, s) : run_bwd<DT, 128, 32>(a, s);
  return dr == 64 ? run_bwd<DT, 64, 64>(a, s) : run_bwd<DT, 64, 32>(a, s);
}

}  // namespace latent

hipError_t launch_latent_bwd(const LatentArgs& a, int dn, int dr, int dt, hipStream_t s) {
  return dt == 0 ? latent::bwd_by_dims<0>(a, dn, dr, s) : dt == 1 ? latent::bwd_by_dims<1>(a, dn, dr, s)
                                                                  : latent::bwd_by_dims<2>(a, dn, dr, s);
}

}  // namespace kda
