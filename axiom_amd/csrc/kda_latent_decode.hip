// Latent attention over the paged cache (absorbed form) and the cache's append.
//
// A cache row holds a token's normed latent (R elements, key and value of every
// head at once) and its rotated key (dr elements): s = scale q . row,
// o = softmax(s) row[:R].

#include "kda_internal.h"
#include "kda_latent.h"

#include <type_traits>

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
// Bound by memory: every element is read and written once, 16 (norm) or 8 bytes a
// lane.  16384 tokens, H16 R512 dr64 bf16: 22 us from a warm cache, 29 to 33 from
// cold memory, 3.3 TB/s (a large copy reaches 5.1; the heads' rotary parts are
// pieces of 128 bytes); one token 2.5 us of kernel.  Loading two or three rounds of
// rotations ahead took 23.2 for 22.4 warm; it was not measured cold.
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
// All sequences' key tiles form one line that is cut into equal runs, one a
// workgroup, so workgroups carry equal work whatever the lengths are; a run
// that covers only part of a sequence leaves its unnormalised sum, maximum and
// row sum for the join kernel.  A workgroup holds 16 or 64 query rows (row =
// token * H + head) in registers; the cache is read once for them.
//
// Up to 16 rows: bound by the cache's bytes (30 flop a byte), so everything else
// stays out of the copies' way.  Four waves score and four add: a score wave
// holds the queries and takes every fourth tile of 16 keys (S^T = K Q^T,
// 16x16x32), an output wave a quarter of the R columns for all tiles (O^T += V^T
// P^T, 16x16x16, V^T being the tile's rows read transposed; the lane that made
// a probability is the lane that needs it).  Tiles pass through a ring of eight
// LDS buffers (147 KB): three on their way, four being scored over four
// intervals, one added; an interval is one barrier.  The one score wave that
// finishes in an interval raises the running maximum, if its tile asks for it,
// so the waves agree on it without an exchange, and nothing is left to merge.
// fp32, with operands twice as large: two score waves and a ring of four.
// 64 sequences of 1 to 8192 tokens, H16 R512 dr64 bf16: 28.8 us with the join, 3.0
// TB/s of the cache's bytes, in fp32 66; one of 512 tokens 12.9 us, a chain of loads.
template <int DT, int R, int DR>
struct DecCfg {
  static constexpr int ES = El<DT>::ES;
  static constexpr int KT = 16;                            // keys of a tile
  static constexpr int SP = ES == 2 ? 4 : 2;               // score waves, and intervals that a tile is scored over
  static constexpr int RING = ES == 2 ? 8 : 4, AHEAD = RING - SP - 1;
  typedef Tile<R, ES> TN;
  typedef Tile<DR, ES> TR;
  static constexpr int OFF_R = TN::bytes(16);
  static constexpr int BUF = OFF_R + TR::bytes(16);
  static constexpr int PN = 16 * TN::CPR / 64, PR = 16 * TR::CPR / 64;   // its 1 KiB pieces
};

// Row fragment of the 16 x 16 x 32 product: lane m = l & 15, group gq = l >> 4;
// element j is column 32 s + 8 gq + j.
template <class TL, class F>
__device__ __forceinline__ F row_frag16(const char* base, int row, int s, int gq) {
  if constexpr (sizeof(F) == 16) {
    return *reinterpret_cast<const F*>(base + TL::off(row, 4 * s, gq));
  } else {
    F f;
    const f4 a = *reinterpret_cast<const f4*>(base + TL::off(row, 8 * s, 2 * gq));
    const f4 b = *reinterpret_cast<const f4*>(base + TL::off(row, 8 * s + 1, 2 * gq));
#pragma unroll
    for (int j = 0; j < 4; ++j) { f[j] = a[j]; f[4 + j] = b[j]; }
    return f;
  }
}
// The lane's four probabilities (keys 4 gq ..) as the second operand of the 16 x 16 x 16 product.
template <int DT> struct P4 { typedef f4 t; };
template <> struct P4<1> { typedef s4v t; };
template <> struct P4<2> { typedef h4 t; };
template <int DT>
__device__ __forceinline__ typename P4<DT>::t to_p4(const float (&p)[4]) {
  if constexpr (DT == 0) return f4{p[0], p[1], p[2], p[3]};
  else if constexpr (DT == 1) return __builtin_bit_cast(s4v, make_uint2(pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3])));
  else return h4{static_cast<_Float16>(p[0]), static_cast<_Float16>(p[1]), static_cast<_Float16>(p[2]), static_cast<_Float16>(p[3])};
}
__device__ __forceinline__ f4 mma_p(f4 c, const f4& a, const f4& b) { return mma16(c, a, b); }
__device__ __forceinline__ f4 mma_p(f4 c, const h4& a, const h4& b) { return mma16(c, a, b); }
__device__ __forceinline__ f4 mma_p(f4 c, const s4v& a, const s4v& b) { return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0); }
// First operand of O^T += V^T P^T: column base + col0 + m of V, keys 4 gq + j; base a
// multiple of 64 (128 in fp32 rows past 256 columns), col0 a constant below it.
template <int DT, class TL>
__device__ __forceinline__ typename P4<DT>::t v_frag(const char* tile, int base, int col0, int lane) {
  const int i = lane & 15, gq = lane >> 4;
  if constexpr (DT == 0) {
    f4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[j] = *reinterpret_cast<const float*>(tile + TL::off(4 * gq + j, (base + col0) >> 2, i >> 2) + 4 * (i & 3));
    return v;
  } else {
    return __builtin_bit_cast(typename P4<DT>::t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s4)(tile + TL::off(4 * gq + (i >> 2), (base + col0) >> 3, (i & 3) >> 1) + 8 * (i & 1))));
  }
}

// Length of sequence b, inside what its table can hold.
__device__ __forceinline__ int seq_len(const LatentDecodeArgs& a, int b) {
  const int64_t cap = static_cast<int64_t>(a.per) << a.page_shift;
  const int n = a.lens[b];
  return n < 0 ? 0 : (n > cap ? static_cast<int>(cap) : n);
}
__device__ __forceinline__ int wave_sum(int n) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) n += __shfl_xor(n, s, 64);
  return __builtin_amdgcn_readfirstlane(n);
}
// inclusive prefix sum over the lanes
__device__ __forceinline__ int wave_scan(int n) {
  const int lane = __lane_id();
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(n, d, 64);
    n += lane >= d ? up : 0;
  }
  return n;
}

// Places of a sequence on the line: its tiles, and a.pad for what a workgroup
// spends on a sequence beside them (queries, first copies, the waves' sums), so
// that one run does not collect many short sequences.
__device__ __forceinline__ int places(const LatentDecodeArgs& a, int len, int KT) {
  return len > 0 ? (len + KT - 1) / KT + a.pad : 0;
}
// The part of the line that workgroup w covers: places [g, g1), the first of them
// place t of sequence b.
struct Run {
  int g, g1, b, t, len;              // len: sequence b's length
  __device__ __forceinline__ Run uniform() const {   // in scalar registers
    return {__builtin_amdgcn_readfirstlane(g), __builtin_amdgcn_readfirstlane(g1), __builtin_amdgcn_readfirstlane(b),
            __builtin_amdgcn_readfirstlane(t), __builtin_amdgcn_readfirstlane(len)};
  }
};
__device__ __forceinline__ Run find_run(const LatentDecodeArgs& a, int w, int KT) {
  const int lane = __lane_id();
  Run r{0, 0, 0, 0, 0};
  if (a.whole) {                     // a workgroup a sequence
    r.b = w;
    r.len = seq_len(a, w);
    r.g1 = (r.len + KT - 1) / KT;
    return r;
  }
  int n = lane < a.B ? seq_len(a, lane) : 0, nt = places(a, n, KT);
  const int first = wave_scan(nt);           // of the first 64 sequences
  int total = __builtin_amdgcn_readlane(first, 63);
  if (a.B > 64) {
    int sum = 0;
    for (int i = lane + 64; i < a.B; i += 64) sum += places(a, seq_len(a, i), KT);
    total += wave_sum(sum);
  }
  const int per = max(a.least, (total + a.wgs - 1) / a.wgs);
  r.g = w * per;
  r.g1 = min(total, r.g + per);
  const bool tell = blockIdx.x == 0 && threadIdx.x < 64;   // the join kernel's starts of the sequences
  if (tell && lane == 0) a.line[0] = per;
  int base = 0;
  bool found = false;
  for (int s0 = 0; s0 < a.B; s0 += 64) {
    if (s0 > 0) {
      n = s0 + lane < a.B ? seq_len(a, s0 + lane) : 0;
      nt = places(a, n, KT);
    }
    const int inc = s0 > 0 ? wave_scan(nt) : first;
    if (tell && s0 + lane < a.B) a.line[1 + s0 + lane] = base + inc - nt;
    const unsigned long long hit = __ballot(base + inc > r.g);
    if (hit && !found) {
      const int x = __ffsll(static_cast<long long>(hit)) - 1;
      r.b = s0 + x;
      r.t = r.g - base - (__builtin_amdgcn_readlane(inc, x) - __builtin_amdgcn_readlane(nt, x));
      r.len = __builtin_amdgcn_readlane(n, x);
      found = true;
    }
    if (found && !tell) break;
    base += __builtin_amdgcn_readlane(inc, 63);
  }
  return r;
}

// workgroup -> run and row group; the groups of one run are eight workgroups
// apart, on one XCD, whose L2 then serves all but the first
__device__ __forceinline__ void run_group(const LatentDecodeArgs& a, int& w, int& grp) {
  if (a.wgs % 8 == 0) {
    grp = (blockIdx.x >> 3) % a.groups;
    w = (blockIdx.x / (8 * a.groups)) * 8 + (blockIdx.x & 7);
  } else {
    grp = blockIdx.x % a.groups;
    w = blockIdx.x / a.groups;
  }
}

// zeros for the rows of an empty sequence
template <int DT, int R>
__device__ __forceinline__ void empty_rows(const LatentDecodeArgs& a, int b, int r0, int r1, int threads) {
  for (int i = threadIdx.x; i < (r1 - r0) * (R / 4); i += threads) {
    const int64_t row = static_cast<int64_t>(b) * a.Tq * a.H + r0 + i / (R / 4);
    store4<DT>(a.o, row * R + 4 * (i % (R / 4)), 0.f, 0.f, 0.f, 0.f);
    if (i % (R / 4) == 0) a.lse[row] = -INFINITY;
  }
}

// Page of this lane's key x of tile j (KT keys): where a page holds a tile or more
// it is the same for all, read by the scalar unit (the table does not change
// under the kernel; a vector load's wait would cover the copies).
template <int KT>
__device__ __forceinline__ int page_of_tile(const LatentDecodeArgs& a, const int32_t* table, int len, int j, int x) {
  if ((1 << a.page_shift) >= KT) {
    const auto* t = (const __attribute__((address_space(4))) int32_t*)table;
    return t[__builtin_amdgcn_readfirstlane(min(j * KT, len - 1) >> a.page_shift)];
  }
  return fresh(table[min(j * KT + x, len - 1) >> a.page_shift]);   // waited for here, not where the branches meet
}
// page of token tok by a vector load
__device__ __forceinline__ int page_of(const LatentDecodeArgs& a, const int32_t* table, int tok) {
  return table[tok >> a.page_shift];
}
// whether tile j begins a page (or holds several)
__device__ __forceinline__ bool new_page(const LatentDecodeArgs& a, int j, int KT) {
  return ((j * KT) & ((1 << a.page_shift) - 1)) == 0 || (1 << a.page_shift) < KT;
}
// cache row of token tok, its page clamped into the cache
__device__ __forceinline__ int slot_of(const LatentDecodeArgs& a, int page, int tok) {
  return (min(max(page, 0), static_cast<int>(a.n_pages - 1)) << a.page_shift) + (tok & ((1 << a.page_shift) - 1));
}

// One 1 KiB piece of a tile's cache rows to LDS: the part of the rows from byte
// `from` on that tile TL holds, TL's first byte at dst.  slot: the cache row of
// key `lane`.  A piece inside one row has its row in scalar registers.  dst: an
// array (the compiler's own copy) or, for copy16_untracked, its LDS address.
__device__ __forceinline__ void put_piece(const char* src, unsigned off, char* dst) { copy16(src + off, dst); }
__device__ __forceinline__ void put_piece(const char* src, unsigned off, unsigned dst) { copy16_untracked(src, off, dst); }
__device__ __forceinline__ void put_piece(const char* src, char* dst) { copy16(src, dst); }
__device__ __forceinline__ void put_piece(const char* src, unsigned dst) { copy16_untracked(src, dst); }
template <class TL, class DST>
__device__ __forceinline__ void copy_piece(const char* cache, int row_bytes, int from, int slot, int piece, int lane, DST dst) {
  if constexpr (TL::CPR % 64 == 0) {
    constexpr int PPR = TL::CPR / 64;      // pieces of a row
    const int r = piece / PPR;
    const char* src = cache + static_cast<int64_t>(__builtin_amdgcn_readlane(slot, r)) * row_bytes + (from + piece % PPR * 1024);
    put_piece(src, static_cast<unsigned>((lane ^ TL::swz(r)) << 4), dst + piece * 1024);
  } else {
    const int r = piece * (64 / TL::CPR) + lane / TL::CPR;
    const char* src = cache + static_cast<int64_t>(__shfl(slot, r, 64)) * row_bytes + (from + (((lane % TL::CPR) ^ TL::swz(r)) << 4));
    put_piece(src, dst + piece * 1024);
  }
}

template <int DT, int R, int DR>
__global__ __launch_bounds__(512) void kda_latent_decode16_kernel(LatentDecodeArgs a) {
  typedef DecCfg<DT, R, DR> C;
  typedef typename El<DT>::frag F;
  typedef typename El<DT>::t E;
  typedef typename P4<DT>::t PV;
  constexpr int ES = C::ES, KT = C::KT, SP = C::SP, RING = C::RING, AHEAD = C::AHEAD;
  constexpr int W = R + DR, KS = W / 32, KSN = R / 32, NV = R / 64;
  constexpr int KP = (KS + (SP > 2 ? SP - 2 : 1)) / (SP > 2 ? SP - 1 : 2);   // products of an interval; SP = 4 keeps the last for the softmax
  constexpr int PW = (C::PN + C::PR) / 8;                       // pieces of a tile that every wave copies at least
  __shared__ __attribute__((aligned(1024))) char buf[RING * C::BUF];
  __shared__ __attribute__((aligned(16))) PV sp[2][64];         // a tile's probabilities, by tile parity
  __shared__ float top[16], fac[2][16], red[2][SP][16];
  __shared__ int rose[2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, gq = lane >> 4;
  const bool scoring = wave < 4;
  int w, grp;
  run_group(a, w, grp);
  Run run = find_run(a, w, KT).uniform();
  const int rows = a.Tq * a.H, r = grp * 16 + m, cr = min(r, rows - 1);
  if (a.whole && run.g1 == 0) empty_rows<DT, R>(a, w, grp * 16, min(rows, grp * 16 + 16), 512);

  const float c = a.scale * kLog2e, lazy = kLazy / c;
  const char* cache = static_cast<const char*>(a.cache);
  const unsigned lds0 = lds_address(buf);

  while (run.g < run.g1) {
    const int b = run.b, len = run.len, n_all = (len + KT - 1) / KT;
    const int ta = run.t, tb = min(n_all, ta + (run.g1 - run.g));   // this segment's tiles
    if (ta < tb) {
    const int32_t* table = a.table + static_cast<int64_t>(b) * a.per;
    auto page_at = [&](int j) { return page_of_tile<KT>(a, table, len, j, m); };
    auto fetch = [&](int j, int page) {
      const int slot = slot_of(a, page, min(j * KT + m, len - 1)), ln = fresh(lane) & 63;
      const unsigned dst = lds0 + (j & (RING - 1)) * C::BUF;
#pragma unroll
      for (int p = wave; p < C::PN + C::PR; p += 8) {
        if (p < C::PN) copy_piece<typename C::TN>(cache, W * ES, 0, slot, p, ln, dst);
        else copy_piece<typename C::TR>(cache, W * ES, R * ES, slot, p - C::PN, ln, dst + C::OFF_R);
      }
    };
    int pages[AHEAD + 1];
#pragma unroll
    for (int x = 0; x <= AHEAD; ++x) pages[x] = page_at(ta + x);
    F q[KS];
    if (wave < SP) {
      const E* qp = static_cast<const E*>(a.q) + (static_cast<int64_t>(b) * rows + cr) * W;
#pragma unroll
      for (int s = 0; s < KS; ++s) q[s] = *reinterpret_cast<const F*>(qp + 32 * s + 8 * gq);
    }
    if (threadIdx.x < 16) top[threadIdx.x] = max_init(c);
#pragma unroll
    for (int x = 0; x < AHEAD; ++x)
      if (ta + x < tb) fetch(ta + x, pages[x]);
    int page = pages[AHEAD];                 // of the next tile to copy
    wait_vmem_all();                         // the queries' wait, which covers the first copies, is this one and no later one

    // interval i: tile i begins to be scored, tile i - SP is added, tile i + AHEAD copied
    auto turn = [&](int i) {
      if (i + AHEAD - 1 < tb) wait_vmem_but<(AHEAD - 1) * PW>();
      else wait_vmem_all();
      lds_barrier();
      if (i + AHEAD < tb) {
        fetch(i + AHEAD, page);
        if (new_page(a, i + AHEAD + 1, KT)) page = page_at(i + AHEAD + 1);
      }
    };
    const bool whole = ta == 0 && tb == n_all;
    const int64_t srow = (static_cast<int64_t>(2 * w + (ta > 0 ? 0 : 1)) * a.groups + grp) * 16;

    if (scoring) {
      const int seen = len - (a.Tq - 1 - cr / a.H);
      float mo = max_init(c), l = 0.f;       // the maximum that l is against
      f4 s0, s1;
      int j = ta + wave;                     // the tile in hand
      auto score = [&](auto phase) {
        constexpr int ph = decltype(phase)::value;
        const char* cur = buf + (j & (RING - 1)) * C::BUF;
        const int ln = fresh(lane), fm = ln & 15, fg = ln >> 4;
        if constexpr (ph == 0) s0 = s1 = f4{0, 0, 0, 0};
        constexpr int k0 = ph * KP, k1 = k0 + KP < KS ? k0 + KP : KS;
        if constexpr (k0 < k1) {
          F kf[k1 - k0];
#pragma unroll
          for (int k = k0; k < k1; ++k)
            kf[k - k0] = k < KSN ? row_frag16<typename C::TN, F>(cur, fm, k, fg)
                                 : row_frag16<typename C::TR, F>(cur + C::OFF_R, fm, k - KSN, fg);
#pragma unroll
          for (int k = k0; k < k1; ++k) {
            if (k & 1) s1 = mma_s(s1, kf[k - k0], q[k]);
            else s0 = mma_s(s0, kf[k - k0], q[k]);
          }
        }
        if constexpr (ph == SP - 1) {
          const int key0 = j * KT + 4 * gq, par = j & 1;
          f4 s = s0 + s1;
#pragma unroll
          for (int e = 0; e < 4; ++e) s[e] = key0 + e < seen ? s[e] : -INFINITY;
          const float tm = group_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
          float mx = top[m];
          const bool up = __any(tm > mx + lazy);
          if (up) {
            const float nm = fmaxf(mx, tm);
            if (gq == 0) {
              fac[par][m] = fast_exp2((mx - nm) * c);
              top[m] = nm;
            }
            mx = nm;
          }
          if (lane == 0) rose[par] = up;
          l *= fast_exp2((mo - mx) * c);
          mo = mx;
          float e[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) e[x] = fast_exp2(fmaf(s[x], c, kLift<DT> - mx * c));
          l += (e[0] + e[1]) + (e[2] + e[3]);
          sp[par][lane] = to_p4<DT>(e);
          j += SP;
        }
      };
      for (int i = ta; i < tb + SP; ++i) {
        turn(i);
        const int ph = i - j;
        if (wave >= SP || j >= tb || ph < 0) continue;
        if (ph == 0) score(std::integral_constant<int, 0>());
        else if (ph == 1) score(std::integral_constant<int, 1>());
        else if constexpr (SP > 2) {
          if (ph == 2) score(std::integral_constant<int, 2>());
          else score(std::integral_constant<int, SP - 1>());
        }
      }
      l = group_sum(l);
      if (wave < SP && gq == 0) {
        red[0][wave][m] = mo;
        red[1][wave][m] = l;
      }
      lds_barrier();
      if (wave == 0 && gq == 0 && r < rows) {
        const float mx = top[m];
        float ls = 0.f;
#pragma unroll
        for (int x = 0; x < SP; ++x) ls = fmaf(fast_exp2((red[0][x][m] - mx) * c), red[1][x][m], ls);
        if (whole) {
          a.lse[static_cast<int64_t>(b) * rows + r] = ls == 0.f ? -INFINITY : (mx * c - kLift<DT> + __log2f(ls)) * kLn2;
        } else {
          a.part_ml[2 * (srow + m)] = mx * c - kLift<DT>;
          a.part_ml[2 * (srow + m) + 1] = ls;
        }
      }
    } else {
      const int col = (wave - 4) * (R / 4);
      f4 acc[NV];
#pragma unroll
      for (int v = 0; v < NV; ++v) acc[v] = f4{0, 0, 0, 0};
      for (int i = ta; i < tb + SP; ++i) {
        turn(i);
        const int j = i - SP;
        if (j < ta) continue;
        const int par = j & 1, up = rose[par];
        const char* cur = buf + (j & (RING - 1)) * C::BUF;
        const int ln = fresh(lane);
        const PV p = sp[par][ln];
        PV vf[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) vf[v] = v_frag<DT, typename C::TN>(cur, col, 16 * v, ln);
        if (__builtin_amdgcn_readfirstlane(up)) {
          const float al = fac[par][m];
#pragma unroll
          for (int v = 0; v < NV; ++v) acc[v] *= al;
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) acc[v] = mma_p(acc[v], vf[v], p);
      }
      lds_barrier();
      float ls = 0.f;
      const float mx = top[m];
#pragma unroll
      for (int x = 0; x < SP; ++x) ls = fmaf(fast_exp2((red[0][x][m] - mx) * c), red[1][x][m], ls);
      if (r < rows) {
        const float inv = ls > 0.f ? 1.f / ls : ls;   // NaN stays NaN
        const int64_t row = static_cast<int64_t>(b) * rows + r;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          if (ls == 0.f) acc[v] = f4{0, 0, 0, 0};     // nothing visible: zeros, whatever 0 times the others' rows made
          const int at = col + 16 * v + 4 * gq;
          if (whole) store4<DT>(a.o, row * R + at, acc[v][0] * inv, acc[v][1] * inv, acc[v][2] * inv, acc[v][3] * inv);
          else *reinterpret_cast<f4*>(a.part_o + (srow + m) * R + at) = acc[v];
        }
      }
    }
    lds_barrier();                           // the sums have been read
    }
    run.g += places(a, len, KT) - ta;
    ++run.b;
    run.t = 0;
    if (run.g < run.g1) run.len = seq_len(a, run.b);
  }
}

// More than 16 rows: 64 a workgroup (16-bit types).  120 flop a byte and more, so
// the tile is shared and the work split by what a wave holds: four waves hold
// the queries (16 rows each, 72 registers) and make a tile's probabilities,
// four hold the output (64 rows by a quarter of the R columns, 128 registers)
// and add the tile before.  The two on a SIMD have about as many products
// (16x16x32 and 32x32x16); one's softmax runs under the other's products, and a
// tile of 32 keys takes one barrier.  A row's keys of a tile are all in one wave,
// so its maximum needs no exchange; where it rises (by 2^8, seldom) the factor
// goes to the output waves beside the probabilities.  Four buffers: one each
// is written to, arrived, scored and added.
// 8 sequences of 20000 to 32768 tokens, two queries each, H64 R512 dr64 fp16: 86 us
// and 9 of join, 650 TFLOP/s; the score waves' LDS reads (each of four reads every
// key) and their chain of reads, products and softmax bound it.  Two waves a tile
// with 32 rows each and 16 keys at a time, which reads LDS half as often, took 112:
// the chain is per tile, not per key.
template <int DT, int R, int DR>
__global__ __launch_bounds__(512) void kda_latent_decode64_kernel(LatentDecodeArgs a) {
  typedef typename El<DT>::frag F;
  typedef typename El<DT>::t E;
  typedef Tile<R, 2> TN;
  typedef Tile<DR, 2> TR;
  constexpr int KT = 32;
  typedef Tile<KT, 2> TP;
  constexpr int W = R + DR, KS = W / 32, KSN = R / 32, NV = R / 128;
  constexpr int OFF_R = TN::bytes(KT), BUF = OFF_R + TR::bytes(KT);
  constexpr int PN = KT * TN::CPR / 64 / 8, PR = KT * TR::CPR / 64;   // pieces: latents a wave; rotary parts in all
  __shared__ __attribute__((aligned(1024))) char buf0[BUF];
  __shared__ __attribute__((aligned(1024))) char buf1[BUF];
  __shared__ __attribute__((aligned(1024))) char buf2[BUF];
  __shared__ __attribute__((aligned(1024))) char buf3[BUF];
  __shared__ __attribute__((aligned(1024))) char sp[2][TP::bytes(64)];   // probabilities, by tile parity
  __shared__ float fac[2][64];               // factor of the rows' sums before this tile
  __shared__ int4 rose[2];                   // whether a score wave's rows have one
  __shared__ float ml[2][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int own = wave & 3;
  const bool scoring = wave < 4;
  int w, grp;
  run_group(a, w, grp);
  Run run = find_run(a, w, KT).uniform();
  const int rows = a.Tq * a.H, r0 = grp * 64;
  if (a.whole && run.g1 == 0) empty_rows<DT, R>(a, w, r0, min(rows, r0 + 64), 512);

  const float c = a.scale * kLog2e, lazy = kLazy / c;
  const char* cache = static_cast<const char*>(a.cache);

  while (run.g < run.g1) {
    const int b = run.b, len = run.len, n_all = (len + KT - 1) / KT;
    const int ta = run.t, tb = min(n_all, ta + (run.g1 - run.g));
    if (ta < tb) {
    const int32_t* table = a.table + static_cast<int64_t>(b) * a.per;
    auto token = [&](int j) { return min(j * KT + (lane & 31), len - 1); };   // a key a lane
    auto fetch = [&](int slot, char* dst) {
      const int ln = fresh(lane) & 63;
#pragma unroll
      for (int p = 0; p < PN; ++p) copy_piece<TN>(cache, W * 2, 0, slot, wave + 8 * p, ln, dst);
      if (wave < PR) copy_piece<TR>(cache, W * 2, R * 2, slot, wave, ln, dst + OFF_R);
    };
    const int tok0 = token(ta), tok1 = token(ta + 1);
    const int page0 = page_of(a, table, tok0), page1 = page_of(a, table, tok1);
    int page = page_of(a, table, token(ta + 2));
    fetch(slot_of(a, page0, tok0), buf0);
    if (ta + 1 < tb) fetch(slot_of(a, page1, tok1), buf1);

    // interval i: tile i is scored, tile i - 1 added, tile i + 2 copied
    auto turn = [&](int i, char* nxt) {
      if (i + 1 < tb) wait_vmem_but<PN>();
      else wait_vmem_all();
      lds_barrier();
      if (i + 2 < tb) {
        const int slot = slot_of(a, page, token(i + 2));
        page = page_of(a, table, token(i + 3));
        fetch(slot, nxt);
      }
    };
    const bool whole = ta == 0 && tb == n_all;
    const int64_t srow = (static_cast<int64_t>(2 * w + (ta > 0 ? 0 : 1)) * a.groups + grp) * 64;

    if (scoring) {
      const int m = lane & 15, gq = lane >> 4, r = min(r0 + 16 * own + m, rows - 1);
      F q[KS];
      {
        const E* qp = static_cast<const E*>(a.q) + (static_cast<int64_t>(b) * rows + r) * W;
#pragma unroll
        for (int s = 0; s < KS; ++s) q[s] = *reinterpret_cast<const F*>(qp + 32 * s + 8 * gq);
      }
      const int seen = len - (a.Tq - 1 - r / a.H);
      const int clear = (len - (a.Tq - 1)) / KT;   // tiles before this one have no masked key
      // the lane's places: of the fragments in a tile (a latent's repeat every four), of its probabilities
      int at[4 + DR / 32], put[2];
#pragma unroll
      for (int k = 0; k < 4 + DR / 32; ++k) at[k] = k < 4 ? TN::off(m, 4 * k, gq) : TR::off(m, 4 * (k - 4), gq);
#pragma unroll
      for (int t = 0; t < 2; ++t) put[t] = TP::off(m, 2 * t, gq & 1, 16 * own) + 8 * (gq >> 1);
      float mx = max_init(c), mc = mx * c - kLift<DT>, l = 0.f;
      auto step = [&](int i, const char* cur, char* nxt) {
        turn(i, nxt);
        f4 s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int t = 0; t < 2; ++t)
            s[t] = mma_s(s[t], *reinterpret_cast<const F*>(cur + (k < KSN ? at[k & 3] + ((k >> 2) * 256 + TN::bytes(16 * t))
                                                                           : at[4 + (k - KSN)] + (OFF_R + TR::bytes(16 * t)))), q[k]);
        pace<2 * KS, 8, 1, 1>();
        __builtin_amdgcn_sched_barrier(0);
        if (i >= clear) {
          const int key0 = i * KT + 4 * gq;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[t][e] = key0 + 16 * t + e < seen ? s[t][e] : -INFINITY;
        }
        float tm = fmaxf(s[0][0], s[1][0]);
#pragma unroll
        for (int e = 1; e < 4; ++e) tm = fmaxf(tm, fmaxf(s[0][e], s[1][e]));
        const bool up = __any(tm > mx + lazy);
        if (up) {
          const float nm = fmaxf(mx, group_max(tm)), al = fast_exp2((mx - nm) * c);
          mx = nm;
          mc = nm * c - kLift<DT>;
          l *= al;
          if (gq == 0) fac[i & 1][16 * own + m] = al;
        }
        if (lane == 0) reinterpret_cast<int*>(&rose[i & 1])[own] = up;
        float sum[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) p[e] = fast_exp2(fmaf(s[t][e], c, -mc));
          sum[t] = (p[0] + p[1]) + (p[2] + p[3]);
          // the output waves' fragment order: chunk 2 t + half, first or second four keys
          store4<DT>(sp[i & 1] + put[t], 0, p[0], p[1], p[2], p[3]);
        }
        l += sum[0] + sum[1];
      };
      for (int i = ta; i < tb;) {
        step(i, buf0, buf2);
        if (++i >= tb) break;
        step(i, buf1, buf3);
        if (++i >= tb) break;
        step(i, buf2, buf0);
        if (++i >= tb) break;
        step(i, buf3, buf1);
        ++i;
      }
      turn(tb, buf0);                        // the last tile is added; nothing to copy
      l = group_sum(l);
      if (gq == 0) {
        ml[0][16 * own + m] = mc;
        ml[1][16 * own + m] = l;
      }
      lds_barrier();
      if (gq == 0 && r0 + 16 * own + m < rows) {
        if (whole) {
          a.lse[static_cast<int64_t>(b) * rows + r] = l == 0.f ? -INFINITY : (mc + __log2f(l)) * kLn2;
        } else {
          a.part_ml[2 * (srow + 16 * own + m)] = mc;
          a.part_ml[2 * (srow + 16 * own + m) + 1] = l;
        }
      }
    } else {
      const int m = lane & 31, h = lane >> 5;
      f16v acc[NV][2];
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[v][n][e] = 0.f;
      // the lane's places: of its columns in a tile, of the probabilities
      int at[NV][2], pat[2];
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int y = 0; y < 2; ++y)
          at[v][y] = TN::off(4 * h + (m >> 2 & 3) + 8 * y, (own * (R / 4) + 32 * v) >> 3, 2 * (m >> 4) + ((m & 3) >> 1)) + 8 * (m & 1);
#pragma unroll
      for (int k = 0; k < 2; ++k) pat[k] = TP::off(m, 2 * k, h);
      auto step = [&](int i, const char* prev, char* nxt) {
        turn(i, nxt);
        const int par = (i - 1) & 1;
        const int4 up = rose[par];
        if (__builtin_amdgcn_readfirstlane(up.x | up.y | up.z | up.w)) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int mine = n == 0 ? (m < 16 ? up.x : up.y) : (m < 16 ? up.z : up.w);
            const float al = mine ? fac[par][32 * n + m] : 1.f;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
              for (int e = 0; e < 16; ++e) acc[v][n][e] *= al;
          }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const F p0 = *reinterpret_cast<const F*>(sp[par] + pat[k]), p1 = *reinterpret_cast<const F*>(sp[par] + pat[k] + TP::bytes(32));
#pragma unroll
          for (int v = 0; v < NV; ++v) {
            union { s4v s[2]; F f; } u;
#pragma unroll
            for (int y = 0; y < 2; ++y)
              u.s[y] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(prev + at[v][y] + TN::bytes(16 * k)));
            const F vf = u.f;
            acc[v][0] = mma(acc[v][0], vf, p0);
            acc[v][1] = mma(acc[v][1], vf, p1);
          }
        }
        __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
        for (int k = 0; k < 2 * NV; ++k) {
          __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      };
      turn(ta, buf2);
      for (int i = ta + 1; i <= tb;) {
        step(i, buf0, buf3);
        if (++i > tb) break;
        step(i, buf1, buf0);
        if (++i > tb) break;
        step(i, buf2, buf1);
        if (++i > tb) break;
        step(i, buf3, buf2);
        ++i;
      }
      lds_barrier();
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int r = r0 + 32 * n + m;
        if (r >= rows) continue;
        const float ls = ml[1][32 * n + m];
        const int64_t row = static_cast<int64_t>(b) * rows + r;
        const int col = own * (R / 4) + 4 * h;
        const float inv = ls > 0.f ? 1.f / ls : ls;   // NaN stays NaN
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f4 o = {acc[v][n][4 * e], acc[v][n][4 * e + 1], acc[v][n][4 * e + 2], acc[v][n][4 * e + 3]};
            if (ls == 0.f) o = f4{0, 0, 0, 0};         // nothing visible: zeros, whatever 0 times the others' rows made
            if (whole) store4<DT>(a.o, row * R + col + 32 * v + 8 * e, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
            else *reinterpret_cast<f4*>(a.part_o + (srow + 32 * n + m) * R + col + 32 * v + 8 * e) = o;
          }
      }
    }
    lds_barrier();                           // the sums have been read
    }
    run.g += places(a, len, KT) - ta;
    ++run.b;
    run.t = 0;
    if (run.g < run.g1) run.len = seq_len(a, run.b);
  }
}

// Joins the parts of a split sequence in run order, one row a workgroup; writes
// the rows of an empty sequence.  Bound by its chain of loads (places of the
// sequence, then the parts): the first eight parts of a half are on their way
// before their factors are known.  Two halves of the workgroup take every second
// part.  4 us for one sequence of 16 rows, 9 for 8 of 128.
template <int DT, int R, int KT>
__global__ __launch_bounds__(R / 2) void kda_latent_join_kernel(LatentDecodeArgs a, int M16) {
  __shared__ float fac[64];
  __shared__ f4 other[R / 4];
  const int rows = a.Tq * a.H, lane = threadIdx.x & 63;
  const int b = blockIdx.y, r = blockIdx.x, half = threadIdx.x / (R / 4), col = (threadIdx.x % (R / 4)) * 4;
  const int per = a.line[0], g0 = a.line[1 + b], n = (seq_len(a, b) + KT - 1) / KT;
  const int64_t row = static_cast<int64_t>(b) * rows + r;
  if (n == 0) {
    if (half == 0) store4<DT>(a.o, row * R + col, 0.f, 0.f, 0.f, 0.f);
    if (threadIdx.x == 0) a.lse[row] = -INFINITY;
    return;
  }
  const int w0 = g0 / per, cnt = (g0 + n - 1) / per - w0 + 1;
  if (cnt == 1) return;
  const int grp = r / M16;
  // part i: run w0 + i, whose first segment began inside the sequence but for part 0
  auto at = [&](int i) {
    return (static_cast<int64_t>(2 * (w0 + i) + (i == 0 ? 1 : 0)) * a.groups + grp) * M16 + (r - grp * M16);
  };
  constexpr int PRE = 8;
  f4 pre[PRE];
#pragma unroll
  for (int x = 0; x < PRE; ++x)
    pre[x] = half + 2 * x < cnt ? *reinterpret_cast<const f4*>(a.part_o + at(half + 2 * x) * R + col) : f4{0, 0, 0, 0};
  float2 ml = lane < cnt ? *reinterpret_cast<const float2*>(a.part_ml + 2 * at(lane)) : make_float2(kMaxInit, 0.f);
  float mx = ml.x;
  for (int i = lane + 64; i < cnt; i += 64) mx = fmaxf(mx, a.part_ml[2 * at(i)]);
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) mx = fmaxf(mx, __shfl_xor(mx, s, 64));
  f4 o = {0, 0, 0, 0};
  float l = 0.f;                             // this lane's parts
  for (int i0 = 0; i0 < cnt; i0 += 64) {
    if (i0 > 0) {
      ml = i0 + lane < cnt ? *reinterpret_cast<const float2*>(a.part_ml + 2 * at(i0 + lane)) : make_float2(kMaxInit, 0.f);
      __syncthreads();
    }
    const float f = i0 + lane < cnt ? fast_exp2(ml.x - mx) : 0.f;
    l = fmaf(f, ml.y, l);
    if (threadIdx.x < 64) fac[lane] = f;
    __syncthreads();
    const int m = min(64, cnt - i0);
    if (i0 == 0) {
#pragma unroll
      for (int x = 0; x < PRE; ++x)
        if (half + 2 * x < m) o += fac[half + 2 * x] * pre[x];
    }
#pragma unroll 8
    for (int i = half + (i0 == 0 ? 2 * PRE : 0); i < m; i += 2)
      o += fac[i] * *reinterpret_cast<const f4*>(a.part_o + at(i0 + i) * R + col);
  }
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) l += __shfl_xor(l, s, 64);
  if (half == 1) other[col / 4] = o;
  __syncthreads();
  if (half == 1) return;
  o += other[col / 4];
  const float inv = l > 0.f ? 1.f / l : l;
  store4<DT>(a.o, row * R + col, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
  if (threadIdx.x == 0) a.lse[row] = l == 0.f ? -INFINITY : (mx + __log2f(l)) * kLn2;
}

template <int DT, int R, int DR>
hipError_t run_append(const LatentAppendArgs& a, hipStream_t s) {
  // few tokens: a workgroup each, so a call of one token is one round of loads;
  // many: a wave each (H16 R512 dr64 bf16 from cold memory, workgroup and wave a
  // token: 1024 tokens 5.8 and 6.7 us, 2048 7.2 and 7.9, 4096 11.7 and 10.8)
  if (a.N <= 2048) kda_latent_append_kernel<DT, R, DR, 4><<<dim3(a.N), dim3(256), 0, s>>>(a);
  else kda_latent_append_kernel<DT, R, DR, 1><<<dim3((a.N + 3) / 4), dim3(256), 0, s>>>(a);
  return hipGetLastError();
}

template <int DT, int R, int DR>
hipError_t run_decode(const LatentDecodeArgs& a, int m_rows, hipStream_t s) {
  if (m_rows == 16) {
    kda_latent_decode16_kernel<DT, R, DR><<<dim3(a.wgs * a.groups), dim3(512), 0, s>>>(a);
  } else if constexpr (DT != 0) {
    kda_latent_decode64_kernel<DT, R, DR><<<dim3(a.wgs * a.groups), dim3(512), 0, s>>>(a);
  } else {
    return hipErrorInvalidValue;
  }
  if (a.whole) return hipGetLastError();
  const dim3 grid(a.Tq * a.H, a.B), block(R / 2);
  if (m_rows == 16) kda_latent_join_kernel<DT, R, 16><<<grid, block, 0, s>>>(a, 16);
  else kda_latent_join_kernel<DT, R, 32><<<grid, block, 0, s>>>(a, 64);
  return hipGetLastError();
}

template <int DT>
hipError_t decode_by_dims(const LatentDecodeArgs& a, int R, int dr, int m_rows, hipStream_t s) {
  if (R == 512) return dr == 64 ? run_decode<DT, 512, 64>(a, m_rows, s) : run_decode<DT, 512, 32>(a, m_rows, s);
  return dr == 64 ? run_decode<DT, 256, 64>(a, m_rows, s) : run_decode<DT, 256, 32>(a, m_rows, s);
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
int latent_decode_tile(int m_rows) { return m_rows == 16 ? 16 : 32; }
hipError_t launch_latent_decode(const LatentDecodeArgs& a, int R, int dr, int dt, int m_rows, hipStream_t s) {
  return dt == 0 ? latent::decode_by_dims<0>(a, R, dr, m_rows, s) : dt == 1 ? latent::decode_by_dims<1>(a, R, dr, m_rows, s)
                                                                        : latent::decode_by_dims<2>(a, R, dr, m_rows, s);
}

}  // namespace kda
