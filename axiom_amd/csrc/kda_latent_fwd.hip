// Latent attention, expanded form, forward: o = softmax(scale (q_n k_n^T + q_r k_r^T)) v.
//
// One pass over the keys with a running maximum and sum.  A workgroup of four
// waves owns 128 queries of one head, a wave 32 of them; key tiles of 64 rows
// (fp32: 32) are copied straight to LDS, the next one while the present one is
// used.  Scores are formed transposed (S^T = K Q^T), so a lane holds one
// query's column: its maximum and sum need one exchange with the lane's other
// half, and the probabilities are the second operand of O^T += V^T P^T in the
// registers they were made in.  The rotary key's tile is read once per head from
// the tensor all heads share; no broadcast copy of it exists anywhere.
// P is rounded to the inputs' type for the second product (the matrix cores'
// operand); the row sum adds the unrounded values.
//
// Bound by the products: B1 H16 T16384, d 128 + 64, bf16, causal takes 1.23 ms,
// 1.12 PFLOP/s over the pairs it has to form (an 8192^3 product reaches 1.19);
// B4 H16 T4096 340 us, 1.01.  128 queries a workgroup and two workgroups a CU,
// because a wave's 32 queries, their output and a score tile are 256 registers.
// fp32 (products 16 times as slow, one workgroup a CU): B1 H8 T1024 39 us.

#include "kda_internal.h"
#include "kda_latent.h"

namespace kda {
namespace latent {

template <int DT, int DN, int DR>
struct FwdCfg {
  static constexpr int ES = El<DT>::ES;
  static constexpr int NW = 4, BM = 32 * NW;
  static constexpr int BN = ES == 2 ? 64 : 32;
  typedef Tile<DN, ES> TN;
  typedef Tile<DR, ES> TR;
  static constexpr int OFF_V = TN::bytes(BN), OFF_R = 2 * TN::bytes(BN);
  static constexpr int BUF = 2 * TN::bytes(BN) + TR::bytes(BN);
};

template <int DT, int DN, int DR>
__global__ __launch_bounds__(256, El<DT>::ES == 2 ? 2 : 1) void kda_latent_fwd_kernel(LatentArgs a, int nqb) {
  typedef FwdCfg<DT, DN, DR> C;
  typedef typename El<DT>::frag F;
  typedef typename El<DT>::t E;
  constexpr int ES = C::ES, BN = C::BN, NB = BN / 32, KN = DN / 16, KR = DR / 16, ND = DN / 32;
  __shared__ __attribute__((aligned(1024))) char buf0[C::BUF];
  __shared__ __attribute__((aligned(1024))) char buf1[C::BUF];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 31, h = lane >> 5;

  Where w;
  int z;
  if (!locate_share(a, nqb, C::BM, BN, true, true, w, z)) return;
  const int b = w.b, head = w.head, q0 = w.r0, qe = w.re, off = w.off, nk = w.ke - w.k0;
  const int row = q0 + wave * 32 + m;         // this lane's query
  const bool live = row < qe;
  const int kmax = a.causal ? min(nk - 1, row + off) : nk - 1;   // last key it sees
  const int wave_lo = a.causal ? min(nk - 1, q0 + wave * 32 + off) : nk - 1;   // last key that all of the wave's queries see
  const int wave_hi = a.causal ? min(nk - 1, min(q0 + wave * 32 + 31, qe - 1) + off) : nk - 1;
  const int blk_hi = a.causal ? min(nk - 1, min(q0 + C::BM - 1, qe - 1) + off) : nk - 1;
  // key tiles of the block (none when no query sees a key) and this workgroup's
  const Share part(max(0, (blk_hi + BN) / BN), a.splits, a.share, z);
  const int nt = part.j1;
  if (z >= part.parts) return;

  F qn[KN], qr[KR];
  {
    const E* qp = static_cast<const E*>(a.q) + b * a.q_b + static_cast<int64_t>(min(row, qe - 1)) * a.q_t + head * a.q_h;
#pragma unroll
    for (int s = 0; s < KN; ++s) qn[s] = *reinterpret_cast<const F*>(qp + 16 * s + 8 * h);
#pragma unroll
    for (int s = 0; s < KR; ++s) qr[s] = *reinterpret_cast<const F*>(qp + DN + 16 * s + 8 * h);
  }

  const char* kvp = static_cast<const char*>(a.kv) + (b * a.kv_b + w.k0 * a.kv_t + head * a.kv_h) * ES;
  const char* krp = static_cast<const char*>(a.kr) + (b * a.kr_b + w.k0 * a.kr_t) * ES;
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
  float mx = max_init(c), mc = mx * c - kLift<DT>, l = 0.f;   // running maximum (raw score units), the exponents' reference, sum
  const float lazy = kLazy / c;
  f16v acc[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[n][i] = 0.f;

  auto step = [&](int j, const char* cur, char* nxt) {
    wait_vmem_all();
    lds_barrier();
    if (j + 1 < nt) fetch(j + 1, nxt);
    const int kt = j * BN;
    if (kt > wave_hi) return;                 // nothing of this tile for this wave's queries
    const int ln = lane, fm = m, fh = h;
    f16v s[NB];
#pragma unroll
    for (int t = 0; t < NB; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[t][i] = 0.f;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < KN; ++k)
#pragma unroll
      for (int t = 0; t < NB; ++t) s[t] = mma(s[t], C::TN::template row_frag<F>(cur, fm, k, fh, 32 * t), qn[k]);
#pragma unroll
    for (int k = 0; k < KR; ++k)
#pragma unroll
      for (int t = 0; t < NB; ++t)
        s[t] = mma(s[t], C::TR::template row_frag<F>(cur + C::OFF_R, fm, k, fh, 32 * t), qr[k]);
    if constexpr (ES == 2) pace<NB * (KN + KR), 6, 1, 1>();
    __builtin_amdgcn_sched_barrier(0);
    if (kt + BN - 1 > wave_lo) {
#pragma unroll
      for (int t = 0; t < NB; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = kt + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3);
          s[t][i] = key <= kmax ? s[t][i] : -INFINITY;
        }
    }
    float tm = s[0][0];
#pragma unroll
    for (int t = 0; t < NB; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) tm = fmaxf(tm, s[t][i]);
    tm = half_max(tm);
    if (__any(tm > mx + lazy)) {
      const float nm = fmaxf(mx, tm);
      const float al = fast_exp2((mx - nm) * c);
      mx = nm;
      mc = nm * c - kLift<DT>;
      l *= al;
#pragma unroll
      for (int n = 0; n < ND; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[n][i] *= al;
    }
    // the tile's sum first: one by one, values below 2^-24 of l would be lost in it
    F pf[2 * NB];
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < 2 * NB; ++u) {
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = fast_exp2(fmaf(s[u >> 1][8 * (u & 1) + e], c, -mc));
        sum += p[e];
      }
      pf[u] = to_frag<DT>(p);
    }
    l += sum;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < 2 * NB; ++u)
#pragma unroll
      for (int n = 0; n < ND; ++n)
        acc[n] = mma(acc[n], C::TN::template col_frag<F>(cur + C::OFF_V, 16 * u, 32 * n, ln), pf[u]);
    if constexpr (ES == 2) pace<2 * NB * ND, 4, 2, 1>();
    __builtin_amdgcn_sched_barrier(0);
  };
  if (part.j0 < nt) fetch(part.j0, buf0);
  for (int j = part.j0; j < nt;) {
    step(j, buf0, buf1);
    if (++j >= nt) break;
    step(j, buf1, buf0);
    ++j;
  }

  l = half_sum(l);
  if (!live) return;
  if (l == 0.f) {   // no visible key: zeros, whatever 0 times the others' values made
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[n][i] = 0.f;
  }
  if (part.parts > 1) {
    const int64_t pr = (static_cast<int64_t>(z) * a.B * a.H + w.bh) * a.Tq + row;
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        store4<0>(a.part, pr * DN + 4 * h + 32 * n + 8 * i, acc[n][4 * i], acc[n][4 * i + 1], acc[n][4 * i + 2], acc[n][4 * i + 3]);
    if (h == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * pr) = make_float2(mc, l);
    return;
  }
  const float inv = l > 0.f ? 1.f / l : l;      // NaN stays NaN
  const int64_t ob = ((static_cast<int64_t>(b) * a.Tq + row) * a.H + head) * DN + 4 * h;
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      store4<DT>(a.o, ob + 32 * n + 8 * i, acc[n][4 * i] * inv, acc[n][4 * i + 1] * inv, acc[n][4 * i + 2] * inv,
                 acc[n][4 * i + 3] * inv);
  if (h == 0) a.lse[static_cast<int64_t>(w.bh) * a.Tq + row] = l == 0.f ? -INFINITY : (mc + __log2f(l)) * kLn2;
}

// Joins the parts of split blocks, in part order; an eighth of a block a workgroup.
// Bound by its launch and one round of loads: 4 to 9 us.
template <int DT, int DN, int DR>
__global__ __launch_bounds__(256) void kda_latent_fwd_join_kernel(LatentArgs a, int nqb) {
  typedef FwdCfg<DT, DN, DR> C;
  constexpr int LPR = DN / 4, RPP = 256 / LPR;
  Where w;
  if (!locate(a, blockIdx.x, nqb, C::BM, true, true, w)) return;
  const int nk = w.ke - w.k0, blk_hi = a.causal ? min(nk - 1, min(w.r0 + C::BM - 1, w.re - 1) + w.off) : nk - 1;
  const int parts = Share(max(0, (blk_hi + C::BN) / C::BN), a.splits, a.share, 0).parts;
  if (parts == 1) return;
  const int col = (threadIdx.x % LPR) * 4;
  const int64_t step = static_cast<int64_t>(a.B) * a.H * a.Tq;
#pragma unroll 2
  for (int r = threadIdx.x / LPR; r < 16; r += RPP) {
    const int row = w.r0 + blockIdx.y * 16 + r;
    if (row >= w.re) break;
    const int64_t pr = static_cast<int64_t>(w.bh) * a.Tq + row;
    float mx = kMaxInit, l = 0.f;
    for (int z = 0; z < parts; ++z) mx = fmaxf(mx, a.part_ml[2 * (z * step + pr)]);
    f4 o = {0, 0, 0, 0};
#pragma unroll 4
    for (int z = 0; z < parts; ++z) {
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (z * step + pr));
      const float f = fast_exp2(ml.x - mx);
      l = fmaf(f, ml.y, l);
      o += f * *reinterpret_cast<const f4*>(a.part + (z * step + pr) * DN + col);
    }
    const float inv = l > 0.f ? 1.f / l : l;
    store4<DT>(a.o, ((static_cast<int64_t>(w.b) * a.Tq + row) * a.H + w.head) * DN + col, o[0] * inv, o[1] * inv, o[2] * inv,
               o[3] * inv);
    if (col == 0) a.lse[pr] = l == 0.f ? -INFINITY : (mx + __log2f(l)) * kLn2;
  }
}

template <int DT, int DN, int DR>
hipError_t run_fwd(const LatentArgs& a, hipStream_t s) {
  constexpr int BM = FwdCfg<DT, DN, DR>::BM;
  // packed: every sequence ends in at most one partial block
  const int64_t nqb = a.cu_q ? static_cast<int64_t>(a.Tq) / BM + a.n_seqs : (static_cast<int64_t>(a.Tq) + BM - 1) / BM;
  const int64_t grid = nqb * a.B * a.H;
  if (grid <= 0) return hipSuccess;
  const unsigned gx = static_cast<unsigned>(grid);
  kda_latent_fwd_kernel<DT, DN, DR><<<a.share > 0 ? dim3(static_cast<unsigned>(a.live * a.B * a.H)) : dim3(gx, a.splits), dim3(256), 0, s>>>(a, static_cast<int>(nqb));
  if (a.splits > 1) kda_latent_fwd_join_kernel<DT, DN, DR><<<dim3(gx, 8), dim3(256), 0, s>>>(a, static_cast<int>(nqb));
  return hipGetLastError();
}

template <int DT>
hipError_t by_dims(const LatentArgs& a, int dn, int dr, hipStream_t s) {
  if (dn == 128) return dr == 64 ? run_fwd<DT, 128, 64>(a, s) : run_fwd<DT, 128, 32>(a, s);
  return dr == 64 ? run_fwd<DT, 64, 64>(a, s) : run_fwd<DT, 64, 32>(a, s);
}

}  // namespace latent

hipError_t launch_latent_fwd(const LatentArgs& a, int dn, int dr, int dt, hipStream_t s) {
  return dt == 0 ? latent::by_dims<0>(a, dn, dr, s) : dt == 1 ? latent::by_dims<1>(a, dn, dr, s) : latent::by_dims<2>(a, dn, dr, s);
}

}  // namespace kda
