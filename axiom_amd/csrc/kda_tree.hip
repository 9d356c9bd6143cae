// KDA states and a tree of drafted tokens: the read-out of every place of a tree
// in one pass over the state, and the state after the path that was accepted.
//
// With gamma_i the product of a = exp(g) over the path of place i and u_j what
// place j writes,
//   S_i = diag(gamma_i) S + sum over j on the path of (gamma_i / gamma_j) k_j u_j^T,
// so the delta rule over a tree is a unit lower triangular system:
//   u_i + beta_i sum_{j above i} L_ij u_j = beta_i (v_i - (gamma_i k_i)^T S),
//   L_ij = k_i . (gamma_i / gamma_j) k_j,
//   o_i = (gamma_i q_i)^T S + sum_{j on the path} A_ij u_j,  A_ij = q_i . (gamma_i / gamma_j) k_j.

#include "kda_common.h"
#include "kda_internal.h"
#include "kda_tree.h"

namespace kda {
namespace {

typedef float f2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f4 mfma4(float a, float b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
template <int N>
__device__ __forceinline__ float row_ror(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + N, 0xF, 0xF, false));
}
// sum over the 16 lanes of a DPP row, in all of them
__device__ __forceinline__ float row_sum16(float x) {
  x += row_ror<8>(x);
  x += row_ror<4>(x);
  x += row_ror<2>(x);
  x += row_ror<1>(x);
  return x;
}
__device__ __forceinline__ float dot4(f4 a, f4 b, float c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = fmaf(a[e], b[e], c);
  return c;
}

// two neighbouring elements, as they lie in memory
template <int DT> struct Two {
  typedef unsigned t;
  static __device__ __forceinline__ f2 floats(unsigned x) {
    if constexpr (DT == 1) return f2{__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u)};
    else return f2{f16bits_to_f32(static_cast<u16>(x)), f16bits_to_f32(static_cast<u16>(x >> 16))};
  }
};
template <> struct Two<0> {
  typedef f2 t;
  static __device__ __forceinline__ f2 floats(f2 x) { return x; }
};

// A float is the sum of three bf16, eight bits each cut off its end: the parts of two floats,
// p0's the largest.  Six of the nine products of two such sums (without the three below 2^-22 of the
// factors' powers of two) are the fp32 product to some 2^-24, at 96 clocks for 256.
struct Parts {
  unsigned p[3];
};
__device__ __forceinline__ Parts parts(float x, float y) {
  Parts r;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const unsigned a = __float_as_uint(x), b = __float_as_uint(y);
    r.p[k] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    x -= __uint_as_float(a & 0xFFFF0000u);
    y -= __uint_as_float(b & 0xFFFF0000u);
  }
  return r;
}
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
// Rows of D fp32 values as planes of NP rows of parts: channel 16 s + 4 g + e at place
// 32 (s / 2) + 8 g + 4 (s % 2) + e, so that the eight of one lane's 16x16x32 operand lie together and a
// float's channels are those the lanes hold of the state.
template <int NP, int LP>
__device__ __forceinline__ void put_parts(u16* planes, int row, int c, int m, f4 v) {
  const Parts a = parts(v[0], v[1]), b = parts(v[2], v[3]);
  u16* at = planes + row * LP + 32 * (2 * c + (m >> 3)) + 8 * (m & 3) + 4 * ((m >> 2) & 1);
#pragma unroll
  for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x2*>(at + k * NP * LP) = u32x2{a.p[k], b.p[k]};
}
struct Split {
  b8 p[3];
};
template <int NP, int LP>
__device__ __forceinline__ Split get_parts(const u16* planes, int row, int at) {
  Split r;
#pragma unroll
  for (int k = 0; k < 3; ++k) r.p[k] = *reinterpret_cast<const b8*>(planes + (k * NP + row) * LP + at);
  return r;
}
constexpr int kPa[6] = {0, 2, 1, 0, 1, 0}, kPb[6] = {2, 0, 1, 1, 0, 0};   // the small products first

// Logarithms along a path are whole numbers of 2^-24: their sums are exact, so gamma_i / gamma_j of two
// places far down a path is as good as their own few decays (a float of 64 or more has steps
// of 2^-17, and a pair's decay would err by those of the whole path before it).  A gate's own
// logarithm is off by 2^-25 whatever its size: what the product with log2 e rounds away is added.
constexpr float kUnits = 16777216.f, kWideGate = 55.f, kLarge = 0x1p40f, kSmall = 0x1p-24f;
constexpr unsigned kWide = 80u << 24;
__device__ __forceinline__ unsigned log2_units(float g) {
  constexpr float low = 1.925963e-8f * kUnits;   // of log2 e, what the float lacks
  g = fminf(fmaxf(g, -64.f), 64.f);              // past kWideGate, and a whole number holds it
  const float t = g * (kLog2e * kUnits), rest = fmaf(g, low, fmaf(g, kLog2e * kUnits, -t));
  return static_cast<unsigned>(static_cast<int>(rintf(t)) + static_cast<int>(rintf(rest)));
}
// 2^x and 2^-x of such a number: only the fraction's powers round
__device__ __forceinline__ void exp2_units(unsigned x, float& up, float& down) {
  const int whole = static_cast<int>(x) >> 24;
  const float part = static_cast<float>(x & 0xFFFFFFu) * (1.f / kUnits);
  up = ldexpf(fast_exp2(part), whole);
  down = ldexpf(fast_exp2(-part), -whole);
}
// bits of |x|: in the order of the values, with infinity and what is no number last
__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// One workgroup a (sequence, head): D / 32 waves of 32 value columns each, whose
// slice of the state waits in registers while the scores are made.
//   1. 16 lanes a place: log2 gamma by doubling along the paths; A and L as products of tiles
//      of gamma_i q_i and k_j / gamma_j (TILES).  Where one channel of one path decays by more than 2^-80 (or
//      grows by as much, or a q or k is very large or small) the whole workgroup takes its pairs one by
//      one instead, the quotient being the product of a over the places between, so that
//      nothing overflows however strong the decay.
//   2. (gamma q)^T S and (gamma k)^T S, the state read once.  Both kinds of products are of
//      fp32 factors in three bf16 parts; as 16x16x4 fp32 products they were 24 us of matrix
//      time for 64 sequences of 32 places and 16 heads, beside 26 of bytes, and the call took 48.
//   3. u tile of 16 places by tile: inverses of the diagonal tiles (I + beta L)^-1 times what the
//      tiles before leave, o from A u, in fp32.  A tile's result is the next product's operand in
//      the registers it was made in (row 4 gq + e of its four is step e's).
// That call takes 41 us (49 if every head has a path past 2^80): the bytes, and phases of the two workgroups of
// a CU that overlap in part (a third does not fit the LDS).  33 to 64 places: 157 KB of LDS and one wave a SIMD, so
// nothing overlaps: B16 chains of 64 29 us and 58 past 2^80, where gates of -0.9 a token bring them; B32 trees 57
// and 88.  Few sequences: a chain of loads, walk, products, 8.4 us for B8 N6 H16.
template <int D, int DT, int NT, bool TILES, int OUT>
__global__ __launch_bounds__(2 * D) void kda_tree_step_kernel(TreeStepArgs a) {
  constexpr int NW = D / 32, NP = 16 * NT, G = 4 * NW, NPG = NP / G > 0 ? NP / G : 1;   // places of a group of 16 lanes
  constexpr int C4 = D / 64, LK = D + 4, LA = NP + 4, LT = 20, LP = D + 8, PL = 3 * NP * LP;
  constexpr int SMALL = 2 * NP * LA + NT * 16 * LT;
  static_assert(2 * PL >= 4 * NP * LK, "what shares a place fits");
  constexpr int THIRD = !TILES ? 0 : PL > 2 * SMALL ? PL : 2 * SMALL;
  __shared__ __attribute__((aligned(16))) u16 pieces[2 * PL + THIRD];
  __shared__ __attribute__((aligned(16))) float small[TILES ? 4 : SMALL];
  u16* const rk = pieces;                // gamma k in parts; on a walk k before
  u16* const rq = pieces + PL;           // gamma q; on a walk a before
  u16* const rn = pieces + 2 * PL;       // log2 gamma; then k / gamma; then A, L, T
  float* const fk = reinterpret_cast<float*>(rk);
  float* const fq = reinterpret_cast<float*>(rq);
  float* const fl = reinterpret_cast<float*>(TILES ? rn : rq);
  float* const As = TILES ? fl : small;
  float* const Ls = As + NP * LA;
  float* const Ts = Ls + NP * LA;
  __shared__ float bet[NP];
  __shared__ int wide[NW];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, gq = lane >> 4, grp = tid >> 4;
  const int b = blockIdx.x / a.H, h = blockIdx.x - b * a.H, N = a.N;
  auto place = [&](int x) { return x * G + ((x & 1) ? G - 1 - grp : grp); };   // deep and shallow ones in turn
  auto token = [&](int i) { return (static_cast<int64_t>(b) * N + min(i, N - 1)) * a.H + h; };

  // the tokens' rows first, then the state: loads return in order
  const int parent = a.parents[static_cast<int64_t>(b) * N + min(lane, N - 1)];
  f4 kv[NPG][C4], qv[NPG][C4], av[NPG][C4];
  float bt[NPG];
#pragma unroll
  for (int x = 0; x < NPG; ++x) {
    const int64_t t = token(place(x));
#pragma unroll
    for (int c = 0; c < C4; ++c) {
      kv[x][c] = ld4<DT>(a.k, t * D + 64 * c + 4 * m);
      qv[x][c] = ld4<DT>(a.q, t * D + 64 * c + 4 * m);
      av[x][c] = ld4<DT>(a.g, t * D + 64 * c + 4 * m);
    }
    bt[x] = ld1<DT>(a.beta, t);
  }
  __builtin_amdgcn_sched_barrier(0);
  const int col = 32 * wave + 2 * m;     // and col + 1: columns m of the wave's two tiles
  const float* Sp = a.state + static_cast<int64_t>(blockIdx.x) * D * D + col;
  f2 S[D / 16][4];
#pragma unroll
  for (int s = 0; s < D / 16; ++s)
#pragma unroll
    for (int e = 0; e < 4; ++e) S[s][e] = *reinterpret_cast<const f2*>(Sp + (16 * s + 4 * gq + e) * D);
  typedef typename Two<DT>::t V2;
  V2 vv[NT][4];                          // v of the lane's rows, its two columns
#pragma unroll
  for (int r = 0; r < NT; ++r)
#pragma unroll
    for (int e = 0; e < 4; ++e) vv[r][e] = static_cast<const V2*>(a.v)[(token(16 * r + 4 * gq + e) * D + col) / 2];
  __builtin_amdgcn_sched_barrier(0);

  const u64 path = tree_paths(parent, N), live = __ballot(path != 0);
  u32x4 lv[NPG][C4];                     // log2 gamma of the places in hand, in units
  unsigned gates = 0, most = 0, least = ~0u;   // |g|; of the largest entries that a lane has of a k and of a scale q
#pragma unroll
  for (int x = 0; x < NPG; ++x) {
    const int i = place(x);
    const bool on = (live >> i) & 1;
    if (!on) bt[x] = 0.f;
#pragma unroll
    for (int c = 0; c < C4; ++c) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        kv[x][c][e] = on ? kv[x][c][e] : 0.f;
        qv[x][c][e] = on ? qv[x][c][e] * a.scale : 0.f;
        av[x][c][e] = on ? av[x][c][e] : 0.f;
        if constexpr (TILES) {
          lv[x][c][e] = log2_units(av[x][c][e]);
          gates = max(gates, abs_bits(av[x][c][e]));
        }
      }
      if constexpr (TILES) *reinterpret_cast<u32x4*>(fl + i * LK + 64 * c + 4 * m) = lv[x][c];
    }
    if constexpr (TILES) {
      float tk = 0.f, tq = 0.f;
#pragma unroll
      for (int c = 0; c < C4; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          tk = fmaxf(tk, fabsf(kv[x][c][e]));
          tq = fmaxf(tq, fabsf(qv[x][c][e]));
        }
      most = max(most, max(__float_as_uint(tk), __float_as_uint(tq)));
      least = min(least, min(__float_as_uint(tk) - 1, __float_as_uint(tq) - 1));   // of zeros only: none
    }
    if (m == 0) bet[i] = bt[x];
  }
  // sums along the paths, their lengths doubling: what a place has plus what the place above its own has
  int up = TILES && path != 0 ? parent : -1;
  while (__any(up >= 0)) {
    u32x4 more[NPG][C4];
    int ui[NPG];
    lds_barrier();
#pragma unroll
    for (int x = 0; x < NPG; ++x) {
      ui[x] = __shfl(up, place(x), 64);
#pragma unroll
      for (int c = 0; c < C4; ++c) more[x][c] = *reinterpret_cast<const u32x4*>(fl + max(ui[x], 0) * LK + 64 * c + 4 * m);
    }
    lds_barrier();
#pragma unroll
    for (int x = 0; x < NPG; ++x) {
      if (ui[x] < 0) continue;
#pragma unroll
      for (int c = 0; c < C4; ++c) {
        lv[x][c] += more[x][c];
        *reinterpret_cast<u32x4*>(fl + place(x) * LK + 64 * c + 4 * m) = lv[x][c];
      }
    }
    const int next = __shfl(up, max(up, 0), 64);
    up = up >= 0 ? next : up;
  }
  // Within 2^80 the quotient may be two factors: gamma_i q_i times k_j / gamma_j, and
  // the scores are products of tiles; past it, or where a gate is not a number, the paths are walked.
  // So they are where q or k is so large that such a factor may overflow (2^40), or so small (2^-24) that
  // its third part may be below 2^-126, which the matrix unit takes for 0: the pair's share need be neither.
  // (Sums that pass 2^128 wrap, but not unseen: the places above have theirs, and a gate is less than
  // the 96 by which one within 80 could reach another such.)
  bool far = !TILES;
  if (TILES) {
    unsigned logs = 0;
#pragma unroll
    for (int x = 0; x < NPG; ++x)
#pragma unroll
      for (int c = 0; c < C4; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) logs = max(logs, lv[x][c][e] + kWide);
    const bool any = __any(logs > 2 * kWide || gates > __float_as_uint(kWideGate) || most > __float_as_uint(kLarge) ||
                           least < __float_as_uint(kSmall) - 1);
    if (lane == 0) wide[wave] = any;
    lds_barrier();
    far = false;
#pragma unroll
    for (int x = 0; x < NW; ++x) far |= wide[x] != 0;
  }
  if (TILES && __builtin_amdgcn_readfirstlane(far) == 0) {
#pragma unroll
    for (int x = 0; x < NPG; ++x) {
#pragma unroll
      for (int c = 0; c < C4; ++c) {
        f4 gm, in;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float up, down;
          exp2_units(lv[x][c][e], up, down);
          gm[e] = up;
          in[e] = down;
        }
        put_parts<NP, LP>(rk, place(x), c, m, gm * kv[x][c]);
        put_parts<NP, LP>(rq, place(x), c, m, gm * qv[x][c]);
        put_parts<NP, LP>(rn, place(x), c, m, in * kv[x][c]);
      }
    }
    lds_barrier();
    // tiles (r, y <= r) of A and of beta L, dealt out to the waves
    constexpr int ITEMS = NT * (NT + 1), MINE = (ITEMS + NW - 1) / NW;
    auto tile = [](int it, int& r, int& y) {
      const int t = it >> 1;
      r = t >= 6 ? 3 : t >= 3 ? 2 : t >= 1 ? 1 : 0;
      y = t - r * (r + 1) / 2;
    };
    f4 sc[MINE];
#pragma unroll
    for (int n = 0; n < MINE; ++n) {
      const int it = wave + n * NW;
      sc[n] = f4{0, 0, 0, 0};
      if (it >= ITEMS) continue;
      int r, y;
      tile(it, r, y);
      f4 s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
#pragma unroll
      for (int p = 0; p < D / 32; ++p) {
        const Split x = get_parts<NP, LP>(it & 1 ? rk : rq, 16 * r + m, 32 * p + 8 * gq);
        const Split z = get_parts<NP, LP>(rn, 16 * y + m, 32 * p + 8 * gq);
#pragma unroll
        for (int k = 0; k < 6; ++k) (p & 1 ? s1 : s0) = mma32_bf16(p & 1 ? s1 : s0, x.p[kPa[k]], z.p[kPb[k]]);
      }
      sc[n] = s0 + s1;
    }
    lds_barrier();                       // k / gamma has been read; the scores go there
#pragma unroll
    for (int n = 0; n < MINE; ++n) {
      const int it = wave + n * NW;
      if (it >= ITEMS) continue;
      int r, y;
      tile(it, r, y);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 16 * r + 4 * gq + e, j = 16 * y + m;
        const bool on = shfl_u64(path, i) >> j & 1;
        if (it & 1) Ls[i * LA + j] = on && j != i ? bet[i] * sc[n][e] : 0.f;
        else As[i * LA + j] = on ? sc[n][e] : 0.f;
      }
    }
  } else {
    for (int i = tid; i < NP * LA / 4; i += 64 * NW) {
      reinterpret_cast<f4*>(As)[i] = f4{0, 0, 0, 0};
      reinterpret_cast<f4*>(Ls)[i] = f4{0, 0, 0, 0};
    }
#pragma unroll
    for (int x = 0; x < NPG; ++x)
#pragma unroll
      for (int c = 0; c < C4; ++c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) av[x][c][e] = fast_exp2(av[x][c][e] * kLog2e);
        *reinterpret_cast<f4*>(fk + place(x) * LK + 64 * c + 4 * m) = kv[x][c];
        *reinterpret_cast<f4*>(fq + place(x) * LK + 64 * c + 4 * m) = av[x][c];
      }
    lds_barrier();
#pragma unroll
    for (int x = 0; x < NPG; ++x) {
      const int i = place(x);
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < C4; ++c) s = dot4(qv[x][c], kv[x][c], s);
      s = row_sum16(s);
      if (m == 0) As[i * LA + i] = s;
      u64 rest = shfl_u64(path, i) & ((u64{1} << i) - 1);   // the places above, the nearest first
      while (__any(rest != 0)) {
        const int j = rest ? 63 - __clzll(static_cast<long long>(rest)) : -1;
        float sq = 0.f, sk = 0.f;
#pragma unroll
        for (int c = 0; c < C4; ++c) {
          const f4 t = av[x][c] * *reinterpret_cast<const f4*>(fk + max(j, 0) * LK + 64 * c + 4 * m);
          const f4 aj = *reinterpret_cast<const f4*>(fq + max(j, 0) * LK + 64 * c + 4 * m);
          sq = dot4(qv[x][c], t, sq);
          sk = dot4(kv[x][c], t, sk);
          if (j >= 0) av[x][c] *= aj;
        }
        sq = row_sum16(sq);
        sk = row_sum16(sk) * bt[x];
        if (j >= 0) {
          if (m < 2) (m == 0 ? As : Ls)[i * LA + j] = m == 0 ? sq : sk;
          rest &= ~(u64{1} << j);
        }
      }
    }
    lds_barrier();
#pragma unroll
    for (int x = 0; x < NPG; ++x) {
#pragma unroll
      for (int c = 0; c < C4; ++c) {
        put_parts<NP, LP>(rk, place(x), c, m, av[x][c] * kv[x][c]);
        put_parts<NP, LP>(rq, place(x), c, m, av[x][c] * qv[x][c]);
      }
    }
  }
  lds_barrier();
  // (I + beta L)^-1 of the diagonal tiles: tile gq, a column a lane, row after row
  if (wave == 0 && gq < NT) {
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == m ? 1.f : 0.f;
#pragma unroll
      for (int k = 0; k < i; ++k) s = fmaf(-Ls[(16 * gq + i) * LA + 16 * gq + k], t[k], s);
      t[i] = s;
      Ts[(gq * 16 + i) * LT + m] = s;
    }
  }

  // Third parts of entries under 2^-102 would be below 2^-126, the matrix unit's 0: a wave whose columns hold
  // nothing of 2^-63 (an exponent with either of its two highest bits) takes 2^64 of them.
  unsigned any = 0;
#pragma unroll
  for (int s = 0; s < D / 16; ++s)
#pragma unroll
    for (int e = 0; e < 4; ++e) any |= __float_as_uint(S[s][e][0]) | __float_as_uint(S[s][e][1]);
  const bool lift = !__any(any & 0x60000000u);
  if (lift) {
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[s][e] *= 0x1p64f;
  }
  f4 pk[NT][2], pq[NT][2];
#pragma unroll
  for (int r = 0; r < NT; ++r)
#pragma unroll
    for (int c = 0; c < 2; ++c) pk[r][c] = pq[r][c] = f4{0, 0, 0, 0};
#pragma unroll
  for (int p = 0; p < D / 32; ++p) {
    Split st[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      u32x4 w[3];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const f2* s = &S[2 * p + (x >> 1)][2 * (x & 1)];
        const Parts two = parts(s[0][c], s[1][c]);
#pragma unroll
        for (int k = 0; k < 3; ++k) w[k][x] = two.p[k];
      }
#pragma unroll
      for (int k = 0; k < 3; ++k) st[c].p[k] = __builtin_bit_cast(b8, w[k]);
    }
#pragma unroll
    for (int r = 0; r < NT; ++r) {
      const Split xk = get_parts<NP, LP>(rk, 16 * r + m, 32 * p + 8 * gq), xq = get_parts<NP, LP>(rq, 16 * r + m, 32 * p + 8 * gq);
#pragma unroll
      for (int k = 0; k < 6; ++k)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          pk[r][c] = mma32_bf16(pk[r][c], xk.p[kPa[k]], st[c].p[kPb[k]]);
          pq[r][c] = mma32_bf16(pq[r][c], xq.p[kPa[k]], st[c].p[kPb[k]]);
        }
    }
  }
  if (lift) {
#pragma unroll
    for (int r = 0; r < NT; ++r)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        pk[r][c] *= 0x1p-64f;
        pq[r][c] *= 0x1p-64f;
      }
  }
  lds_barrier();                         // the inverses are there
  f4 u[NT][2];
#pragma unroll
  for (int r = 0; r < NT; ++r) {
    f4 w[2];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = 16 * r + 4 * gq + e;
      const float be = bet[i];
      const bool on = (live >> i) & 1;
      const f2 v = Two<DT>::floats(vv[r][e]);
#pragma unroll
      for (int c = 0; c < 2; ++c) w[c][e] = on ? be * (v[c] - pk[r][c][e]) : 0.f;
    }
#pragma unroll
    for (int y = 0; y < r; ++y) {
      const f4 l = *reinterpret_cast<const f4*>(Ls + (16 * r + m) * LA + 16 * y + 4 * gq);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int c = 0; c < 2; ++c) w[c] = mfma4(-l[e], u[y][c][e], w[c]);
    }
    const f4 ti = *reinterpret_cast<const f4*>(Ts + (16 * r + m) * LT + 4 * gq);
    u[r][0] = u[r][1] = f4{0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int c = 0; c < 2; ++c) u[r][c] = mfma4(ti[e], w[c][e], u[r][c]);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (!((live >> (16 * r + 4 * gq + e)) & 1)) u[r][0][e] = u[r][1][e] = 0.f;
#pragma unroll
    for (int y = 0; y <= r; ++y) {
      const f4 p = *reinterpret_cast<const f4*>(As + (16 * r + m) * LA + 16 * y + 4 * gq);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int c = 0; c < 2; ++c) pq[r][c] = mfma4(p[e], u[y][c][e], pq[r][c]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = 16 * r + 4 * gq + e;
      if (i >= N) continue;
      const int64_t t = token(i) * D + col;
      const bool on = (live >> i) & 1;
      *reinterpret_cast<f2*>(a.u + t) = f2{u[r][0][e], u[r][1][e]};
      const float x = on ? pq[r][0][e] : 0.f, y = on ? pq[r][1][e] : 0.f;
      if constexpr (OUT == 0) *reinterpret_cast<f2*>(static_cast<float*>(a.o) + t) = f2{x, y};
      else *reinterpret_cast<unsigned*>(static_cast<u16*>(a.o) + t) = pack_bf16x2(x, y);
    }
  }
}

// The state after the path of place last[b], in place: two workgroups a (sequence,
// head), each half of the value columns.  A thread holds four columns of D / 16
// channels; the path's decayed keys go through LDS, the newest 16 places first.  Bound by the
// state's bytes, read and written once: 64 sequences of 16 heads, trees of 32 places, 31.2 us, 4.5 TB/s.
// A place's k and g are waited for before the next one's are asked for (the first time behind the state's
// loads), then u two places at a time: one sequence 3.6 us for a path of two places, its launch, but
// 5.4 for eight, 13.7 for 32 and 24.6 for 64; 16 sequences of 64 45.
template <int D, int DT>
__global__ __launch_bounds__(2 * D) void kda_tree_commit_kernel(TreeCommitArgs a) {
  constexpr int W = D / 2, NCQ = W / 4, RPT = D / 16, PIECE = 16;
  static_assert(2 * D / NCQ * RPT == D && RPT % 4 == 0, "four channels a read");
  __shared__ __attribute__((aligned(16))) float lk[PIECE][D];
  __shared__ __attribute__((aligned(16))) float gam[D];
  const int tid = threadIdx.x, lane = tid & 63, N = a.N;
  const int bh = blockIdx.x >> 1, b = bh / a.H, h = bh - b * a.H, c0 = (blockIdx.x & 1) * W;
  const int last = a.last[b], parent = a.parents[static_cast<int64_t>(b) * N + min(lane, N - 1)];
  if (last < 0 || last >= N) return;
  u64 path = uniform_u64(shfl_u64(tree_paths(parent, N), last));
  if (path == 0) return;
  const int cq = tid % NCQ, d0 = tid / NCQ * RPT;
  float* S = a.state + static_cast<int64_t>(bh) * D * D + c0 + 4 * cq;
  f4 sv[RPT], acc[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    sv[i] = *reinterpret_cast<const f4*>(S + (d0 + i) * D);
    acc[i] = f4{0, 0, 0, 0};
  }
  float fade = 1.f;                      // of channel tid: the product of a over the places behind
  while (path) {
    u64 rest = path;
    int n = 0;
    for (; n < PIECE && rest; ++n) {
      const int j = 63 - __clzll(static_cast<long long>(rest));
      rest &= ~(u64{1} << j);
      if (tid < D) {
        const int64_t t = ((static_cast<int64_t>(b) * N + j) * a.H + h) * D + tid;
        lk[n][tid] = fade * ld1<DT>(a.k, t);
        fade *= fast_exp2(ld1<DT>(a.g, t) * kLog2e);
      }
    }
    if (tid < D && rest == 0) gam[tid] = fade;
    lds_barrier();
    for (int x = 0; x < n; ++x) {
      const int j = 63 - __clzll(static_cast<long long>(path));
      path &= ~(u64{1} << j);
      const f4 uj = *reinterpret_cast<const f4*>(a.u + ((static_cast<int64_t>(b) * N + j) * a.H + h) * D + c0 + 4 * cq);
#pragma unroll
      for (int i = 0; i < RPT; i += 4) {
        const f4 w = *reinterpret_cast<const f4*>(&lk[x][d0 + i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i + e] += w[e] * uj;
      }
    }
    if (path) lds_barrier();             // the piece has been read
  }
#pragma unroll
  for (int i = 0; i < RPT; ++i) *reinterpret_cast<f4*>(S + (d0 + i) * D) = gam[d0 + i] * sv[i] + acc[i];
}

template <int D, int DT, int NT, bool TILES>
hipError_t step_out(const TreeStepArgs& a, int out, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.B * a.H)), block(2 * D);
  if (out == 0) kda_tree_step_kernel<D, DT, NT, TILES, 0><<<grid, block, 0, s>>>(a);
  else kda_tree_step_kernel<D, DT, NT, TILES, 1><<<grid, block, 0, s>>>(a);
  return hipGetLastError();
}
template <int D, int DT>
hipError_t step_places(const TreeStepArgs& a, int out, hipStream_t s) {
  // Paths of up to eight places are walked: B8 N6 8.4 us and 9.0 with products, B64 N8 20.2 and 23.9; a
  // chain of 16 (B4) 11.2 and 9.4, B32 N12 14.7 and 14.7, 32 places (B64) 48.4 and 40.6.
  if (a.N <= 8) return step_out<D, DT, 1, false>(a, out, s);
  if (a.N <= 16) return step_out<D, DT, 1, true>(a, out, s);
  return a.N <= 32 ? step_out<D, DT, 2, true>(a, out, s) : step_out<D, DT, 4, true>(a, out, s);
}
template <int D>
hipError_t step_types(const TreeStepArgs& a, int dt, int out, hipStream_t s) {
  return dt == 0 ? step_places<D, 0>(a, out, s) : dt == 1 ? step_places<D, 1>(a, out, s) : step_places<D, 2>(a, out, s);
}
template <int D>
hipError_t commit_types(const TreeCommitArgs& a, int dt, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(2 * a.B * a.H));
  if (dt == 0) kda_tree_commit_kernel<D, 0><<<grid, dim3(2 * D), 0, s>>>(a);
  else if (dt == 1) kda_tree_commit_kernel<D, 1><<<grid, dim3(2 * D), 0, s>>>(a);
  else kda_tree_commit_kernel<D, 2><<<grid, dim3(2 * D), 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_tree_step(const TreeStepArgs& a, int d, int dt, int out_dt, hipStream_t s) {
  return d == 128 ? step_types<128>(a, dt, out_dt, s) : step_types<64>(a, dt, out_dt, s);
}
hipError_t launch_tree_commit(const TreeCommitArgs& a, int d, int dt, hipStream_t s) {
  return d == 128 ? commit_types<128>(a, dt, s) : commit_types<64>(a, dt, s);
}

}  // namespace kda
