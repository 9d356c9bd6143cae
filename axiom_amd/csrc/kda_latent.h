// Device helpers of the latent-attention kernels (gfx950 / CDNA4 only).
//
// The kernels work on 32 x 32 score tiles (v_mfma_f32_32x32x16, fp32: eight
// v_mfma_f32_32x32x2 on the same registers).  Lane l of a wave has m = l & 31
// and half h = l >> 5; an operand fragment is 8 elements of a 16-wide
// contraction block, and the accumulator's 16 values of a lane are rows
// 8 (i >> 2) + 4 h + (i & 3), i = 0..15, of column m.  Two fragment orders:
//   * row fragment (contraction along a row): element j is column 8 h + j;
//   * column fragment (contraction over rows): element j is row
//     8 (j >> 2) + 4 h + (j & 3), the accumulator's own row order, so a score
//     tile (or its adjoint) is the second operand of the next product with
//     no exchange between lanes, and the first operand is read with its rows
//     transposed (ds_read_b64_tr_b16: a group of 16 lanes reads 4 rows of 16
//     columns and each lane gets one column).
//
// LDS tiles are row-major without padding, because direct global->LDS copies
// write 1 KiB of consecutive bytes per wave instruction; bank conflicts are
// kept out by a permutation of the 16-byte chunks inside each row instead
// (chunk c of row r sits at c ^ swz(r)), applied to the copies' source
// addresses.  A 16-byte read takes 16 lanes at a time, lanes 0-3, 12-15, 20-27 of
// 32 and then the others, an 8-byte one 32: swz gives each such set, of 16
// or 32 rows a fragment and of transposed reads of 4 rows, different banks
// (measured: 37 % of the LDS cycles were conflicts with a permutation that was
// distinct over 8 consecutive rows only).
#pragma once

#include "kda_common.h"
#include "kda_internal.h"

namespace kda {
namespace latent {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4v* lds_s4;

constexpr float kLn2 = 0.6931471805599453f;
// finite start of the running maximum: exp2 of a masked (-inf) score minus it is 0
constexpr float kMaxInit = -1e30f;
// ... in raw score units, where c is the scale times log2 e: times c it has to stay finite too
__device__ __forceinline__ float max_init(float c) { return fmaxf(kMaxInit, -1e37f / c); }
// The running maximum is raised (and the accumulators rescaled) only when a
// tile exceeds it by more than 2^kLazy: probabilities then reach at most
// 2^8, in range for the 16-bit operands and without loss, since the row sum is
// kept in fp32 and both are divided at the end.
constexpr float kLazy = 8.f;
// fp16 probabilities are held 2^7 times as large, up to 2^15: its smallest step, 6e-8, is
// then 5e-10 of the row's maximum, and a hundred thousand keys that are each far below
// it keep what they add up to.  The reference of the exponents is lower by as much.
template <int DT> constexpr float kLift = DT == 2 ? 7.f : 0.f;

template <int DT> struct El;
template <> struct El<0> { typedef float t; typedef f8 frag; static constexpr int ES = 4; };
template <> struct El<1> { typedef u16 t; typedef b8 frag; static constexpr int ES = 2; };
template <> struct El<2> { typedef u16 t; typedef h8 frag; static constexpr int ES = 2; };

__device__ __forceinline__ f16v mma(f16v c, const f8& a, const f8& b) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ f16v mma(f16v c, const b8& a, const b8& b) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f16v mma(f16v c, const h8& a, const h8& b) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// the 16 x 16 forms (32-wide contraction; same fragment rules with four lane groups)
__device__ __forceinline__ f4 mma_s(f4 c, const f8& a, const f8& b) { return mma32(c, a, b); }
__device__ __forceinline__ f4 mma_s(f4 c, const b8& a, const b8& b) { return mma32_bf16(c, a, b); }
__device__ __forceinline__ f4 mma_s(f4 c, const h8& a, const h8& b) { return mma32(c, a, b); }

// eight fp32 values to a fragment (round to nearest even)
template <int DT>
__device__ __forceinline__ typename El<DT>::frag to_frag(const float (&x)[8]) {
  typename El<DT>::frag r;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (DT == 0) r[j] = x[j];
    else if constexpr (DT == 1) r[j] = static_cast<__bf16>(x[j]);
    else r[j] = static_cast<_Float16>(x[j]);
  }
  return r;
}

// four fp32 values to four consecutive elements of global memory
template <int DT>
__device__ __forceinline__ void store4(void* p, int64_t i, float a, float b, float c, float d) {
  if constexpr (DT == 0) {
    *reinterpret_cast<f4*>(static_cast<float*>(p) + i) = f4{a, b, c, d};
  } else if constexpr (DT == 1) {
    *reinterpret_cast<uint2*>(static_cast<u16*>(p) + i) = make_uint2(pack_bf16x2(a, b), pack_bf16x2(c, d));
  } else {
    const h4 v = {static_cast<_Float16>(a), static_cast<_Float16>(b), static_cast<_Float16>(c), static_cast<_Float16>(d)};
    *reinterpret_cast<uint2*>(static_cast<u16*>(p) + i) = __builtin_bit_cast(uint2, v);
  }
}

// x, of which the compiler knows nothing: addresses derived from it inside a loop
// are formed there (a few integer instructions) instead of being held in dozens
// of registers across it, which the accumulators need
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Order of a product's instructions, from here up to the last barrier of the
// scheduler: the reads of AHEAD fragments (RPF LDS reads each) first, then MPF
// products for each further fragment read, then the rest.
template <int N, int AHEAD, int RPF, int MPF>
__device__ __forceinline__ void pace() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * RPF, 0);
#pragma unroll
  for (int i = 0; i < N - AHEAD; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, MPF, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, RPF, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, AHEAD * MPF, 0);
}

// all but the newest N vector memory operations of the wave are done
template <int N>
__device__ __forceinline__ void wait_vmem_but() {
  static_assert(N >= 0 && N < 64, "vmcnt is six bits");
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

// A barrier between LDS reads whose values have been used and writes to their
// places: it waits for nothing.  lds_barrier would wait for the copies on their way
// too, which are LDS writes to the compiler.
__device__ __forceinline__ void reuse_barrier() { asm volatile("s_barrier" : : : "memory"); }

// value combined over the two halves of the wave (lane l and l ^ 32)
__device__ __forceinline__ float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// maximum over the four 16-lane groups
__device__ __forceinline__ float group_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float group_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Direct global->LDS copy of 16 or 4 bytes a lane, to 64 consecutive places from
// dst on (wave-uniform).
__device__ __forceinline__ void copy16(const char* src, char* dst) { __builtin_amdgcn_global_load_lds(src, dst, 16, 0, 0); }
__device__ __forceinline__ void copy4(const void* src, char* dst) { __builtin_amdgcn_global_load_lds(src, dst, 4, 0, 0); }

// The 16-byte copy as an instruction the compiler does not see as a memory access:
// base + off (a lane's) to 1 KiB of LDS from byte address lds on.  The compiler
// makes an LDS read wait for every copy it knows of unless it can tell their
// arrays apart; code with a ring of buffers, indexed while it runs, copies with
// this, waits with wait_vmem_but / wait_vmem_all and a barrier, and has no vector
// loads of its own meanwhile (the compiler's wait for one would cover the copies).
__device__ __forceinline__ void copy16_untracked(const char* base, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void copy16_untracked(const char* src, unsigned lds) {   // a lane's own address
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ unsigned lds_address(const void* p) {
  return static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)p));
}

// An LDS tile of rows of W elements of ES bytes.
template <int W, int ES>
struct Tile {
  static constexpr int RB = W * ES;       // bytes of a row
  static constexpr int CPR = RB / 16;     // 16-byte chunks of a row
  static_assert(RB % 64 == 0, "whole groups of chunks");
  // the permutation stays inside aligned groups of SWZ + 1 chunks
  static constexpr int SWZ = CPR % 16 == 0 ? 15 : CPR % 8 == 0 ? 7 : 3;
  static __device__ __forceinline__ int swz(int r) {
    const int lo = (((r >> 2) ^ (r >> 3)) & 1) << 1 | ((r >> 3) & 1);
    if constexpr (SWZ == 15) return ((r & 3) << 2) | lo;
    else if constexpr (SWZ == 7) return ((r & 2) << 1) | lo;   // two rows per 256 bytes
    else return lo;                                            // four
  }
  // byte offset of chunk cc + cl of row r0 + r: r0 (a multiple of 16) and cc are
  // the parts that unrolling makes constants, r and cl the lane's (cl in bits
  // that cc has clear), so that what the constants add outside the permutation
  // goes into the instruction's offset field
  static __device__ __forceinline__ int off(int r, int cc, int cl = 0, int r0 = 0) {
    return r0 * RB + ((cc & ~SWZ) << 4) + (r * RB + ((((cc & SWZ) | cl) ^ swz(r)) << 4));
  }
  static constexpr int bytes(int rows) { return rows * RB; }

  // row fragment of contraction block ks: row r0 + row, elements 16 ks + 8 h ..
  template <class F>
  static __device__ __forceinline__ F row_frag(const char* base, int row, int ks, int h, int r0 = 0) {
    if constexpr (ES == 2) {
      return *reinterpret_cast<const F*>(base + off(row, 2 * ks, h, r0));
    } else {
      F f;
      const f4 a = *reinterpret_cast<const f4*>(base + off(row, 4 * ks, 2 * h, r0));
      const f4 b = *reinterpret_cast<const f4*>(base + off(row, 4 * ks + 1, 2 * h, r0));
#pragma unroll
      for (int j = 0; j < 4; ++j) { f[j] = a[j]; f[4 + j] = b[j]; }
      return f;
    }
  }
  // column fragment: column col0 + m, rows row0 + 8 (j >> 2) + 4 h + (j & 3)
  template <class F>
  static __device__ __forceinline__ F col_frag(const char* base, int row0, int col0, int lane) {
    if constexpr (ES == 2) {
      const int g = lane >> 4, i = lane & 15;
      const int r = 4 * (g >> 1) + (i >> 2);
      const int cc = col0 >> 3, cl = 2 * (g & 1) + ((i & 3) >> 1);
      const int sub = 8 * (i & 1);
      union { s4v s[2]; F f; } u;
      u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(base + off(r, cc, cl, row0) + sub));
      u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(base + off(r + 8, cc, cl, row0) + sub));
      return u.f;
    } else {
      const int m = lane & 31, h = lane >> 5;
      const int cc = col0 >> 2, cl = m >> 2, sub = (m & 3) * 4;
      F f;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        f[j] = *reinterpret_cast<const float*>(base + off(8 * (j >> 2) + 4 * h + (j & 3), cc, cl, row0) + sub);
      return f;
    }
  }
};

// Direct global->LDS copy of ROWS rows into a tile by NW waves: the wave's
// share of 1 KiB pieces.  Rows past `last` repeat row `last` (a row the mask
// already excludes reads no memory outside the tensor).
template <class TL, int ROWS, int NW>
struct Copy {
  static constexpr int PIECES = ROWS * TL::CPR / 64, RPP = 64 / TL::CPR > 0 ? 64 / TL::CPR : 1;
  static constexpr int PER = (PIECES + NW - 1) / NW;
  static_assert(ROWS * TL::CPR % 64 == 0 && (PIECES % NW == 0 || PIECES < NW), "whole pieces, a share a wave");
  // the permutation repeats every 16 rows: where a wave's pieces are that far
  // apart, one offset a lane serves all of them
  static constexpr bool ONE = RPP * NW % 16 == 0;
  static __device__ __forceinline__ unsigned offset(int p, int wave, int lane, unsigned row_bytes, int last) {
    const int s = (wave + p * NW) * 64 + lane;
    const int r = s / TL::CPR, c = (s % TL::CPR) ^ TL::swz(r);
    return static_cast<unsigned>(min(r, last)) * row_bytes + c * 16;
  }
  unsigned offs[ONE ? 1 : PER];
  __device__ __forceinline__ void init(int wave, int lane, unsigned row_bytes) {
#pragma unroll
    for (int p = 0; p < (ONE ? 1 : PER); ++p) offs[p] = offset(p, wave, lane, row_bytes, ROWS);
  }
  // all rows there; src: the tile's first row (wave-uniform)
  __device__ __forceinline__ void issue(const char* src, char* dst, int wave, unsigned row_bytes) const {
    if (PIECES < NW && wave >= PIECES) return;
    unsigned o = 0;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      if (p == 0 || !ONE) o = static_cast<unsigned>(fresh(static_cast<int>(offs[p])));   // scalar base, 32-bit lane offset
      copy16((ONE ? src + static_cast<size_t>(p * RPP * NW) * row_bytes : src) + o, dst + (wave + p * NW) * 1024);
    }
  }
  // the sequence's last rows
  static __device__ __forceinline__ void issue_last(const char* src, char* dst, int wave, int lane, unsigned row_bytes, int last) {
    if (PIECES < NW && wave >= PIECES) return;
    const int ln = fresh(lane);
#pragma unroll
    for (int p = 0; p < PER; ++p) copy16(src + offset(p, wave, ln, row_bytes, last), dst + (wave + p * NW) * 1024);
  }
};

// A block's share z of its n tiles along the other axis: [j0, j1) of `parts`
// shares of `len` tiles, or (len 0) of `splits` equal ones of at least two.
struct Share {
  int j0, j1, parts;
  __device__ __forceinline__ Share(int n, int splits, int len, int z) {
    const int c = len > 0 ? len : splits > 1 ? max(2, (n + splits - 1) / splits) : max(n, 1);
    parts = max(1, (n + c - 1) / c);
    j0 = z * c;
    j1 = min(n, j0 + c);
  }
};

// The sequence and block of a workgroup.  Dense: block `id` of one batch
// element.  Packed (cu non-null): blocks are numbered sequence by sequence,
// ceil(len / BLK) of each; found by the wave, 64 sequences at a time.  Offsets
// are clamped into [0, T] and made non-decreasing pairwise, so no access
// leaves the tensors whatever they hold.
struct Span { int seq, blk, a, e; };   // rows [a, e) of the packed axis
__device__ __forceinline__ bool find_span(const int32_t* cu, int n_seqs, int T, int BLK, int id, Span& s) {
  const int lane = __lane_id();
  int base = 0;
  for (int s0 = 0; s0 < n_seqs; s0 += 64) {
    const int i = s0 + lane;
    int a = 0, e = 0;
    if (i < n_seqs) {
      a = min(max(cu[i], 0), T);
      e = min(max(cu[i + 1], a), T);
    }
    const int nb = (e - a + BLK - 1) / BLK;
    int inc = nb;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(inc, d, 64);
      inc += lane >= d ? up : 0;
    }
    const unsigned long long hit = __ballot(base + inc > id);
    if (hit) {
      const int w = __ffsll(static_cast<long long>(hit)) - 1;
      s.seq = s0 + w;
      s.blk = __builtin_amdgcn_readfirstlane(id - base - (__shfl(inc, w, 64) - __shfl(nb, w, 64)));
      s.a = __builtin_amdgcn_readfirstlane(__shfl(a, w, 64));
      s.e = __builtin_amdgcn_readfirstlane(__shfl(e, w, 64));
      return true;
    }
    base += __builtin_amdgcn_readfirstlane(__shfl(inc, 63, 64));
  }
  return false;
}

struct Where { int b, head, bh, blk, r0, re, k0, ke, off; };   // rows owned from r0 to re, the other side k0 to ke
// q_side: the workgroup owns queries, else keys.  off: owned query row i sees the
// keys of the sequence with index <= i + off; owned key row j is seen by the
// queries of the sequence with index >= j + off.
// Heads are spread over the eight XCDs (consecutive workgroups go round them), so
// that one XCD's L2 serves a head's rows; reverse: the last block of a head
// first (the one with the longest causal walk).  A causal call takes an XCD's
// heads up to four at a time, the longest blocks of all four first: head by head,
// the last head's longest blocks began when the other heads' were done (B4 H16
// T4096: forward 368 -> 341 us, query pass 658 -> 597, key pass 813 -> 802).  A
// head of 256 blocks is long enough alone.
__device__ __forceinline__ void order(const LatentArgs& a, int id, int nb, bool reverse, int& bh, int& blk) {
  const int bh_n = a.B * a.H;
  if (bh_n % 8 == 0) {
    const int slot = id >> 3, group = a.causal ? max(1, min(4, 256 / nb)) : 1;
    const int g = slot / (nb * group), in = min(group, (bh_n >> 3) - g * group);
    const int i = slot - g * nb * group;
    bh = (id & 7) + 8 * (g * group + i % in);
    blk = i / in;
  } else {
    bh = id % bh_n;
    blk = id / bh_n;
  }
  if (reverse) blk = nb - 1 - blk;
}
// Share `id` of a grid of live shares: heads go round the XCDs, a head's blocks
// follow each other with all their shares.  BN: rows of a tile.
__device__ __forceinline__ void live_share(const LatentArgs& a, int id, int nb, int BN, bool q_side, int len, int& bh, int& blk, int& z) {
  const int bh_n = a.B * a.H, lane = __lane_id(), all = ((q_side ? a.Tk : a.Tq) + BN - 1) / BN, u = id / bh_n;
  bh = id - u * bh_n;
  blk = z = 0;
  for (int b0 = 0, base = 0; b0 < nb; b0 += 64) {
    const int i = b0 + lane;
    int n = all;
    if (a.causal) {
      n = q_side ? max(0, min(a.Tk - 1, min(128 * i + 127, a.Tq - 1) + a.Tk - a.Tq) + BN) / BN
                 : max(0, all - max(0, 128 * i + a.Tq - a.Tk) / BN);
    }
    n = i < nb ? max(1, (n + len - 1) / len) : 0;
    int inc = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(inc, d, 64);
      inc += lane >= d ? up : 0;
    }
    const unsigned long long hit = __ballot(base + inc > u);
    if (hit) {
      const int x = __ffsll(static_cast<long long>(hit)) - 1;
      blk = b0 + x;
      z = u - base - (__builtin_amdgcn_readlane(inc, x) - __builtin_amdgcn_readlane(n, x));
      return;
    }
    base += __builtin_amdgcn_readlane(inc, 63);
  }
}
// Where block blk of head bh stands; false: a packed call's surplus block.
__device__ __forceinline__ bool place(const LatentArgs& a, int bh, int blk, int BM, bool q_side, Where& w) {
  w.bh = bh;
  w.blk = blk;
  w.b = w.bh / a.H;
  w.head = w.bh - w.b * a.H;
  if (a.cu_q) {
    Span s;
    if (!find_span(q_side ? a.cu_q : a.cu_k, a.n_seqs, q_side ? a.Tq : a.Tk, BM, blk, s)) return false;
    const int32_t* o = q_side ? a.cu_k : a.cu_q;
    const int T = q_side ? a.Tk : a.Tq;
    w.r0 = s.a + s.blk * BM;
    w.re = s.e;
    w.k0 = min(max(o[s.seq], 0), T);
    w.ke = min(max(o[s.seq + 1], w.k0), T);
    const int nr = s.e - s.a, no = w.ke - w.k0;
    w.off = no - nr - s.a;   // keys - queries, or queries - keys
  } else {
    w.r0 = blk * BM;
    w.re = q_side ? a.Tq : a.Tk;
    w.k0 = 0;
    w.ke = q_side ? a.Tk : a.Tq;
    w.off = q_side ? a.Tk - a.Tq : a.Tq - a.Tk;
  }
  return true;
}

__device__ __forceinline__ bool locate(const LatentArgs& a, int id, int nb, int BM, bool q_side, bool reverse, Where& w) {
  int bh, blk;
  order(a, id, nb, reverse, bh, blk);
  return place(a, bh, blk, BM, q_side, w);
}
// ... of this workgroup of a pass, and its share z
__device__ __forceinline__ bool locate_share(const LatentArgs& a, int nb, int BM, int BN, bool q_side, bool reverse, Where& w, int& z) {
  const int len = q_side ? a.share : a.share_k;
  int bh, blk;
  z = blockIdx.y;
  if (len > 0) live_share(a, blockIdx.x, nb, BN, q_side, len, bh, blk, z);
  else order(a, blockIdx.x, nb, reverse, bh, blk);
  return place(a, bh, blk, BM, q_side, w);
}

}  // namespace latent
}  // namespace kda
