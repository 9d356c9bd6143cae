// Latent attention over the paged cache (absorbed form) and the cache's append.
//
// A cache row holds a token's normed latent (R elements, key and value of every
// head at once) and its rotated key (dr elements): s = scale q . row,
// o = softmax(s) row[:R].

#include "kda_internal.h"
#include "kda_latent.h"

namespace kda {
namespace latent {

// ------------------------------------------------------------------ append
// Rotation of four pairs: elements i .. i + 3 with i + dr/2 .. (split halves), or
// eight consecutive elements as four neighbouring pairs.
template <int DT, int DR>
__device__ __forceinline__ void rotate_unit(const void* src, int64_t si, void* dst, int64_t di, const float* cs, int u,
                                            bool inter) {
  const int e0 = inter ? 8 * u : 4 * u, e1 = inter ? e0 + 4 : e0 + DR / 2;
  const f4 x = ld4<DT>(src, si + e0), y = ld4<DT>(src, si + e1);
  const f4 c = *reinterpret_cast<const f4*>(cs + 4 * u), s = *reinterpret_cast<const f4*>(cs + DR / 2 + 4 * u);
  const f4 a = inter ? f4{x[0], x[2], y[0], y[2]} : x, b = inter ? f4{x[1], x[3], y[1], y[3]} : y;
  f4 p, q;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    p[e] = a[e] * c[e] - b[e] * s[e];
    q[e] = b[e] * c[e] + a[e] * s[e];
  }
  const f4 o0 = inter ? f4{p[0], q[0], p[1], q[1]} : p, o1 = inter ? f4{p[2], q[2], p[3], q[3]} : q;
  store4<DT>(dst, di + e0, o0[0], o0[1], o0[2], o0[3]);
  store4<DT>(dst, di + e1, o1[0], o1[1], o1[2], o1[3]);
}

// One token by TPW threads' worth of waves: wave 0 of the token norms and stores
// its latent, all of them share the rotations (the row's own and H heads').
// Bound by memory: every element is read and written once, 16 (norm) or 8 bytes a lane.
template <int DT, int R, int DR, int WPT>
__global__ __launch_bounds__(256) void kda_latent_append_kernel(LatentAppendArgs a) {
  constexpr int V = R / 64;               // latent elements of a lane
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int n = blockIdx.x * (4 / WPT) + wv / WPT, part = wv % WPT;
  if (n >= a.N) return;
  const int64_t slot = a.slots[n], pos = min(max(a.positions[n], static_cast<int64_t>(0)), a.P - 1);
  const bool keep = slot >= 0 && slot < a.n_slots;
  const float* cs = a.cos_sin + pos * DR;
  const int64_t src = static_cast<int64_t>(n) * a.rows_t, dst = slot * (R + DR);
  if (part == 0 && keep) {
    f4 x[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) x[i] = ld4<DT>(a.rows, src + lane * V + 4 * i);
    f4 w[V / 4];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      if (a.w) w[i] = *reinterpret_cast<const f4*>(a.w + lane * V + 4 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) ss = fmaf(x[i][e], x[i][e], ss);
    }
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) ss += __shfl_xor(ss, s, 64);
    const float inv = rsqrtf(ss / R + a.eps);
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      f4 y = x[i];
      if (a.w) y = x[i] * inv * w[i];
      store4<DT>(a.cache, dst + lane * V + 4 * i, y[0], y[1], y[2], y[3]);
    }
  }
  constexpr int U = DR / 8;               // rotation units of a head
  const int units = a.q ? (a.H + 1) * U : U;
  for (int i = part * 64 + lane; i < units; i += 64 * WPT) {
    const int hd = i / U - 1, u = i % U;
    if (hd < 0) {
      if (keep) rotate_unit<DT, DR>(a.rows, src + R, a.cache, dst + R, cs, u, a.interleaved);
    } else {
      rotate_unit<DT, DR>(a.q, n * a.q_t + hd * a.q_h, a.q_out, n * a.qo_t + hd * a.qo_h, cs, u, a.interleaved);
    }
  }
}

// ------------------------------------------------------------------ decode
// A workgroup of four waves holds a group of 16 NB query rows (row = token *
// H + head) of one sequence and walks a run of key tiles.  All sequences'
// tiles form one line that is cut into equal runs, so workgroups carry equal
// work whatever the lengths are; a run that covers only part of a sequence
// leaves its unnormalised sum, maximum and row sum for the join kernel.
// The cache is read once per row group: a tile's rows go straight to LDS and
// serve as keys (rows) and as values (the same rows transposed).
// Waves share the tile: for the scores a wave takes 16 keys, for the output a
// quarter of the R columns; the probabilities cross through LDS.
template <int DT, int R, int DR, int NB>
struct DecCfg {
  static constexpr int ES = El<DT>::ES;
  static constexpr int KT = ES == 2 ? 64 : 32;
  typedef Tile<R, ES> TN;
  typedef Tile<DR, ES> TR;
  typedef Tile<KT, ES> TP;
  static constexpr int OFF_R = TN::bytes(KT);
  static constexpr int BUF = OFF_R + TR::bytes(KT);
};

// Fragments of the 16 x 16 products: lane m = l & 15, group gq = l >> 4; element
// j is contraction index 32 s + 8 gq + j.
template <class TL, class F>
__device__ __forceinline__ F row_frag16(const char* base, int row, int s, int gq) {
  if constexpr (sizeof(F) == 16) {
    return *reinterpret_cast<const F*>(base + TL::off(row, 4 * s + gq));
  } else {
    F f;
    const f4 a = *reinterpret_cast<const f4*>(base + TL::off(row, 8 * s + 2 * gq));
    const f4 b = *reinterpret_cast<const f4*>(base + TL::off(row, 8 * s + 2 * gq + 1));
#pragma unroll
    for (int j = 0; j < 4; ++j) { f[j] = a[j]; f[4 + j] = b[j]; }
    return f;
  }
}
template <class TL, class F>
__device__ __forceinline__ F col_frag16(const char* base, int s, int col0, int lane) {
  if constexpr (sizeof(F) == 16) {
    const int i = lane & 15, r = 32 * s + 8 * (lane >> 4) + (i >> 2);
    const int c = (col0 >> 3) + ((i & 3) >> 1), sub = 8 * (i & 1);
    union { s4v v[2]; F f; } u;
    u.v[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(base + TL::off(r, c) + sub));
    u.v[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(base + TL::off(r + 4, c) + sub));
    return u.f;
  } else {
    const int m = lane & 15, r = 32 * s + 8 * (lane >> 4);
    const int c = (col0 + m) >> 2, sub = ((col0 + m) & 3) * 4;
    F f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = *reinterpret_cast<const float*>(base + TL::off(r + j, c) + sub);
    return f;
  }
}

// Length of sequence b, inside what its table can hold.
__device__ __forceinline__ int seq_len(const LatentDecodeArgs& a, int b) {
  const int64_t cap = static_cast<int64_t>(a.per) << a.page_shift;
  const int n = a.lens[b];
  return n < 0 ? 0 : (n > cap ? static_cast<int>(cap) : n);
}
// Tiles of sequences [0, b1), summed by the wave.
template <int KT>
__device__ __forceinline__ int tiles_before(const LatentDecodeArgs& a, int b1) {
  int n = 0;
  for (int i = __lane_id(); i < b1; i += 64) n += (seq_len(a, i) + KT - 1) / KT;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) n += __shfl_xor(n, s, 64);
  return __builtin_amdgcn_readfirstlane(n);
}

template <int DT, int R, int DR, int NB>
__global__ __launch_bounds__(256, 1) void kda_latent_decode_kernel(LatentDecodeArgs a) {
  typedef DecCfg<DT, R, DR, NB> C;
  typedef typename El<DT>::frag F;
  typedef typename El<DT>::t E;
  constexpr int ES = C::ES, KT = C::KT, W = R + DR, KS = W / 32, KSN = R / 32, NV = R / 64, M16 = 16 * NB;
  __shared__ __attribute__((aligned(1024))) char buf0[C::BUF];
  __shared__ __attribute__((aligned(1024))) char buf1[C::BUF];
  __shared__ __attribute__((aligned(1024))) char sp[C::TP::bytes(M16)];
  __shared__ float red[4][M16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, gq = lane >> 4;

  // the row groups of one run are eight workgroups apart, on one XCD, whose L2 serves the second
  int w, grp;
  if (a.wgs % 8 == 0) {
    grp = (blockIdx.x >> 3) % a.groups;
    w = (blockIdx.x / (8 * a.groups)) * 8 + (blockIdx.x & 7);
  } else {
    grp = blockIdx.x % a.groups;
    w = blockIdx.x / a.groups;
  }
  const int total = tiles_before<KT>(a, a.B);
  const int per = (total + a.wgs - 1) / a.wgs;
  int g = w * per;
  const int g1 = min(total, g + per);
  if (g >= g1) return;
  // sequence and tile of the run's first tile
  int b = 0, t = 0;
  {
    int base = 0;
    for (int s0 = 0; s0 < a.B; s0 += 64) {
      const int nt_ = s0 + lane < a.B ? (seq_len(a, s0 + lane) + KT - 1) / KT : 0;
      int inc = nt_;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int up = __shfl_up(inc, d, 64);
        inc += lane >= d ? up : 0;
      }
      const unsigned long long hit = __ballot(base + inc > g);
      if (hit) {
        const int x = __ffsll(static_cast<long long>(hit)) - 1;
        b = s0 + x;
        t = __builtin_amdgcn_readfirstlane(g - base - (__shfl(inc, x, 64) - __shfl(nt_, x, 64)));
        break;
      }
      base += __builtin_amdgcn_readfirstlane(__shfl(inc, 63, 64));
    }
  }

  const int rows = a.Tq * a.H;
  const float c = a.scale * kLog2e, lazy = kLazy / c;
  const char* cache = static_cast<const char*>(a.cache);

  while (g < g1) {
    const int len = seq_len(a, b), n_all = (len + KT - 1) / KT;
    if (n_all == 0) { ++b; t = 0; continue; }
    const int ta = t, tb = min(n_all, t + (g1 - g));   // this segment's tiles
    const int32_t* table = a.table + static_cast<int64_t>(b) * a.per;

    // cache row of this lane's key of a tile (KT <= 64 keys, one a lane)
    auto slot_of = [&](int j) {
      const int tok = min(j * KT + (lane & (KT - 1)), len - 1);
      const int page = min(max(table[tok >> a.page_shift], 0), static_cast<int>(a.n_pages - 1));
      return (page << a.page_shift) + (tok & ((1 << a.page_shift) - 1));
    };
    auto fetch = [&](int slot, char* dst) {
      constexpr int PN = KT * C::TN::CPR / 64, PR = KT * C::TR::CPR / 64;
#pragma unroll
      for (int p = 0; p < PN / 4; ++p) {
        const int s = (wave + 4 * p) * 64 + lane, r = s / C::TN::CPR;
        const char* src = cache + static_cast<int64_t>(__shfl(slot, r, 64)) * (W * ES) + (((s % C::TN::CPR) ^ C::TN::swz(r)) << 4);
        copy16(src, dst + (wave + 4 * p) * 1024);
      }
#pragma unroll
      for (int p = 0; p < (PR + 3) / 4; ++p) {
        if (PR % 4 != 0 && wave + 4 * p >= PR) break;
        const int s = (wave + 4 * p) * 64 + lane, r = s / C::TR::CPR;
        const char* src = cache + static_cast<int64_t>(__shfl(slot, r, 64)) * (W * ES) + R * ES +
                          (((s % C::TR::CPR) ^ C::TR::swz(r)) << 4);
        copy16(src, dst + C::OFF_R + (wave + 4 * p) * 1024);
      }
    };

    int next_slot = slot_of(ta);
    // queries of the group: lane column m of each 16-row block
    F q[NB][KS];
    int seen[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int r = min(grp * M16 + 16 * n + m, rows - 1);
      seen[n] = len - (a.Tq - 1 - r / a.H);
      const E* qp = static_cast<const E*>(a.q) + (static_cast<int64_t>(b) * rows + r) * W;
#pragma unroll
      for (int s = 0; s < KS; ++s) q[n][s] = *reinterpret_cast<const F*>(qp + 32 * s + 8 * gq);
    }
    lds_barrier();                          // the last segment's reads of the buffers are done
    fetch(next_slot, buf0);
    if (ta + 1 < tb) next_slot = slot_of(ta + 1);

    f4 acc[NB][NV];
    float mx[NB], mc[NB], l[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      mx[n] = kMaxInit;
      mc[n] = kMaxInit * c;
      l[n] = 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v) acc[n][v] = f4{0, 0, 0, 0};
    }

    auto step = [&](int j, const char* cur, char* nxt) {
      wait_vmem_all();
      lds_barrier();
      if (j + 1 < tb) {
        fetch(next_slot, nxt);
        if (j + 2 < tb) next_slot = slot_of(j + 2);
      }
      f4 s[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n) s[n] = f4{0, 0, 0, 0};
      if (16 * wave < KT) {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const F kf = k < KSN ? row_frag16<typename C::TN, F>(cur, 16 * wave + m, k, gq)
                               : row_frag16<typename C::TR, F>(cur + C::OFF_R, 16 * wave + m, k - KSN, gq);
#pragma unroll
          for (int n = 0; n < NB; ++n) s[n] = mma_s(s[n], kf, q[n][k]);
        }
        const int key0 = j * KT + 16 * wave + 4 * gq;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][i] = key0 + i < seen[n] ? s[n][i] : -INFINITY;
          float tm = fmaxf(fmaxf(s[n][0], s[n][1]), fmaxf(s[n][2], s[n][3]));
          tm = fmaxf(tm, __shfl_xor(tm, 16, 64));
          tm = fmaxf(tm, __shfl_xor(tm, 32, 64));
          if (gq == 0) red[wave][16 * n + m] = tm;
        }
      }
      lds_barrier();
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        float tm = red[0][16 * n + m];
#pragma unroll
        for (int x = 1; x < KT / 16; ++x) tm = fmaxf(tm, red[x][16 * n + m]);
        if (__any(tm > mx[n] + lazy)) {
          const float nm = fmaxf(mx[n], tm), al = fast_exp2((mx[n] - nm) * c);
          mx[n] = nm;
          mc[n] = nm * c;
          l[n] *= al;
#pragma unroll
          for (int v = 0; v < NV; ++v) acc[n][v] *= al;
        }
        if (16 * wave < KT) {
          float p[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[i] = fast_exp2(fmaf(s[n][i], c, -mc[n]));
            l[n] += p[i];
          }
          const int key = 16 * wave + 4 * gq;
          store4<DT>(sp + C::TP::off(16 * n + m, key * ES / 16) + (key * ES) % 16, 0, p[0], p[1], p[2], p[3]);
        }
      }
      lds_barrier();
#pragma unroll
      for (int k = 0; k < KT / 32; ++k) {
        F pf[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) pf[n] = row_frag16<typename C::TP, F>(sp, 16 * n + m, k, gq);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const F vf = col_frag16<typename C::TN, F>(cur, k, wave * (R / 4) + 16 * v, lane);
#pragma unroll
          for (int n = 0; n < NB; ++n) acc[n][v] = mma_s(acc[n][v], vf, pf[n]);
        }
      }
    };
    for (int j = ta; j < tb;) {
      step(j, buf0, buf1);
      if (++j >= tb) break;
      step(j, buf1, buf0);
      ++j;
    }

    // row sums over the four lane groups and the four waves
    lds_barrier();
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      l[n] += __shfl_xor(l[n], 16, 64);
      l[n] += __shfl_xor(l[n], 32, 64);
      if (gq == 0) red[wave][16 * n + m] = l[n];
    }
    lds_barrier();
    const bool whole = ta == 0 && tb == n_all;
    const int64_t slot = (static_cast<int64_t>(2 * w + (ta > 0 ? 0 : 1)) * a.groups + grp) * M16;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int r = grp * M16 + 16 * n + m;
      const float ls = red[0][16 * n + m] + red[1][16 * n + m] + red[2][16 * n + m] + red[3][16 * n + m];
      if (r < rows) {
        const int64_t row = static_cast<int64_t>(b) * rows + r;
        const int col = wave * (R / 4) + 4 * gq;
        if (whole) {
          const float inv = ls > 0.f ? 1.f / ls : ls;   // nothing visible: zeros; NaN stays NaN
#pragma unroll
          for (int v = 0; v < NV; ++v)
            store4<DT>(a.o, row * R + col + 16 * v, acc[n][v][0] * inv, acc[n][v][1] * inv, acc[n][v][2] * inv,
                       acc[n][v][3] * inv);
          if (wave == 0 && gq == 0) a.lse[row] = ls == 0.f ? -INFINITY : (mc[n] + __log2f(ls)) * kLn2;
        } else {
          const int64_t sr = slot + 16 * n + m;
#pragma unroll
          for (int v = 0; v < NV; ++v) *reinterpret_cast<f4*>(a.part_o + sr * R + col + 16 * v) = acc[n][v];
          if (wave == 0 && gq == 0) {
            a.part_ml[2 * sr] = mc[n];
            a.part_ml[2 * sr + 1] = ls;
          }
        }
      }
    }
    g += tb - ta;
    ++b;
    t = 0;
  }
}

// Joins the parts of a split sequence in run order; writes the rows of a sequence of length zero.
template <int DT, int R, int KT>
__global__ __launch_bounds__(256) void kda_latent_join_kernel(LatentDecodeArgs a, int M16) {
  constexpr int TPR = R / 4, RPB = 256 / TPR;
  const int rows = a.Tq * a.H;
  const int b = blockIdx.y, r = blockIdx.x * RPB + threadIdx.x / TPR, col = (threadIdx.x % TPR) * 4;
  const int n = (seq_len(a, b) + KT - 1) / KT;
  const int g0 = tiles_before<KT>(a, b), total = tiles_before<KT>(a, a.B);
  if (r >= rows) return;
  const int64_t row = static_cast<int64_t>(b) * rows + r;
  if (n == 0) {
    store4<DT>(a.o, row * R + col, 0.f, 0.f, 0.f, 0.f);
    if (col == 0) a.lse[row] = -INFINITY;
    return;
  }
  const int per = (total + a.wgs - 1) / a.wgs;
  const int w0 = g0 / per, w1 = (g0 + n - 1) / per;
  if (w0 == w1) return;
  const int grp = r / M16;
  auto at = [&](int w) { return (static_cast<int64_t>(2 * w + (w == w0 ? 1 : 0)) * a.groups + grp) * M16 + (r - grp * M16); };
  float mx = kMaxInit;
  for (int w = w0; w <= w1; ++w) mx = fmaxf(mx, a.part_ml[2 * at(w)]);
  f4 o = {0, 0, 0, 0};
  float l = 0.f;
  for (int w = w0; w <= w1; ++w) {
    const int64_t s = at(w);
    const float f = fast_exp2(a.part_ml[2 * s] - mx);
    l = fmaf(f, a.part_ml[2 * s + 1], l);
    o += f * *reinterpret_cast<const f4*>(a.part_o + s * R + col);
  }
  const float inv = l > 0.f ? 1.f / l : l;
  store4<DT>(a.o, row * R + col, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
  if (col == 0) a.lse[row] = l == 0.f ? -INFINITY : (mx + __log2f(l)) * kLn2;
}

template <int DT, int R, int DR>
hipError_t run_append(const LatentAppendArgs& a, hipStream_t s) {
  // few tokens: a workgroup each, so a call of one token is one round of loads;
  // many: a wave each
  if (a.N < 1024) kda_latent_append_kernel<DT, R, DR, 4><<<dim3(a.N), dim3(256), 0, s>>>(a);
  else kda_latent_append_kernel<DT, R, DR, 1><<<dim3((a.N + 3) / 4), dim3(256), 0, s>>>(a);
  return hipGetLastError();
}

template <int DT, int R, int DR, int NB>
hipError_t run_decode(const LatentDecodeArgs& a, hipStream_t s) {
  kda_latent_decode_kernel<DT, R, DR, NB><<<dim3(a.wgs * a.groups), dim3(256), 0, s>>>(a);
  constexpr int RPB = 256 / (R / 4);
  kda_latent_join_kernel<DT, R, DecCfg<DT, R, DR, NB>::KT>
      <<<dim3((a.Tq * a.H + RPB - 1) / RPB, a.B), dim3(256), 0, s>>>(a, 16 * NB);
  return hipGetLastError();
}

template <int DT, int R, int DR>
hipError_t decode_by_rows(const LatentDecodeArgs& a, int nb, hipStream_t s) {
  if (nb == 1) return run_decode<DT, R, DR, 1>(a, s);
  if (nb == 2) return run_decode<DT, R, DR, 2>(a, s);
  if constexpr (DT != 0) return run_decode<DT, R, DR, 4>(a, s);
  return hipErrorInvalidValue;
}

template <int DT>
hipError_t decode_by_dims(const LatentDecodeArgs& a, int R, int dr, int nb, hipStream_t s) {
  if (R == 512) return dr == 64 ? decode_by_rows<DT, 512, 64>(a, nb, s) : decode_by_rows<DT, 512, 32>(a, nb, s);
  return dr == 64 ? decode_by_rows<DT, 256, 64>(a, nb, s) : decode_by_rows<DT, 256, 32>(a, nb, s);
}
template <int DT>
hipError_t append_by_dims(const LatentAppendArgs& a, int R, int dr, hipStream_t s) {
  if (R == 512) return dr == 64 ? run_append<DT, 512, 64>(a, s) : run_append<DT, 512, 32>(a, s);
  return dr == 64 ? run_append<DT, 256, 64>(a, s) : run_append<DT, 256, 32>(a, s);
}

}  // namespace latent

hipError_t launch_latent_append(const LatentAppendArgs& a, int R, int dr, int dt, hipStream_t s) {
  return dt == 0 ? latent::append_by_dims<0>(a, R, dr, s) : dt == 1 ? latent::append_by_dims<1>(a, R, dr, s)
                                                                    : latent::append_by_dims<2>(a, R, dr, s);
}
hipError_t launch_latent_decode(const LatentDecodeArgs& a, int R, int dr, int dt, int nb, hipStream_t s) {
  return dt == 0 ? latent::decode_by_dims<0>(a, R, dr, nb, s) : dt == 1 ? latent::decode_by_dims<1>(a, R, dr, nb, s)
                                                                        : latent::decode_by_dims<2>(a, R, dr, nb, s);
}

}  // namespace kda
