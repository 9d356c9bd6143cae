// Verification of a tree of drafted tokens against the target's distributions, from
// given random numbers (include/tree_mi355x.h): the walk from the sequence's end
// down the tree, and the token that follows.
//
// A decision compares 24-bit numbers' products and sums over a vocabulary; all of
// that is in 64 bits, so another order of the same sums decides alike but for one
// case in 2^40 or so.  Bound by rows: one of the target and of each draft refused for the next
// token, and the same for every sibling asked after a refusal, since Z is a sum over the
// vocabulary; the walk itself needs a few entries of the rows, a lane a place.  64 sequences
// of 16 places and 128000 fp32 entries: 52 us, of which a pass over one pair of rows of all
// is 13 of bytes, two to three are needed in turn (a place has three children at most), and 7 are the
// second launch.  R is not kept: after its k-th refusal among siblings a workgroup reads the target's row and
// k of draft's, all of them whole, so k refused siblings cost k^2 / 2 rows one after the other.  Every child refused, 128000
// fp32 entries, B1 and B64: 3 children 45 and 120 us, 8 220 and 685, 24 1.8 and 3.9 ms, 64 (B1) 12 ms.  Without
// draft Z needs no row: 64 sequences of 16 places as trees 17 us, as stars 30.

#include "kda_internal.h"
#include "kda_tree.h"

// products and differences round by themselves, as the definition has them
#pragma clang fp contract(off)

namespace kda {
namespace {

constexpr int kWaves = 16, kThreads = 64 * kWaves;

// EPL elements of a row at any alignment: one 16-byte load
template <int DT> struct Pack { static constexpr int EPL = DT == 0 ? 4 : 8; };
template <int DT>
__device__ __forceinline__ u32x4 load_pack(const void* row, int64_t at) {
  u32x4 x;
  __builtin_memcpy(&x, static_cast<const char*>(row) + at * (DT == 0 ? 4 : 2), 16);
  return x;
}
template <int DT>
__device__ __forceinline__ float element(const u32x4& x, int e) {
  if constexpr (DT == 0) return __uint_as_float(x[e]);
  else if constexpr (DT == 1) return __uint_as_float(e & 1 ? x[e >> 1] & 0xFFFF0000u : x[e >> 1] << 16);
  else return f16bits_to_f32(static_cast<u16>(e & 1 ? x[e >> 1] >> 16 : x[e >> 1]));
}
__device__ __forceinline__ double readlane_f64(double x, int lane) {
  const u64 b = __builtin_bit_cast(u64, x);
  const unsigned lo = __builtin_amdgcn_readlane(static_cast<int>(b), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), lane);
  return __builtin_bit_cast(double, static_cast<u64>(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) x += __shfl_xor(x, s, 64);
  return x;
}
__device__ __forceinline__ double wave_scan(double x) {
  const int lane = __lane_id();
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double up = __shfl_up(x, d, 64);
    x += lane >= d ? up : 0.0;
  }
  return x;
}

// The weights R that the next token is drawn from: row `cur` + 1 of the target, less
// what the rejected children (bits) took of it.
struct Weights {
  const void* p;
  const void* draft;      // the sequence's
  int64_t d_row;
  u64 rej;
};
// lane i: the Z that child i was asked with, and its token
template <int DT, bool DRAFT>
__device__ __forceinline__ double weight(const Weights& w, double z, int x, int v) {
  const float p = ld1<DT>(w.p, v);
  double r = p > 0.f ? p : 0.0;
  for (u64 rest = w.rej; rest; rest &= rest - 1) {
    const int i = __ffsll(static_cast<long long>(rest)) - 1;
    if constexpr (DRAFT) r = fmax(r - readlane_f64(z, i) * static_cast<double>(ld1<DT>(w.draft, i * w.d_row + v)), 0.0);
    else r = v == __builtin_amdgcn_readlane(x, i) ? 0.0 : r;
  }
  return r;
}
// The wave's sums of R and (PLAIN) of the row itself over entries [lo, hi), a lane's share.
template <int DT, bool DRAFT, bool PLAIN>
__device__ __forceinline__ void sum_range(const Weights& w, double z, int x, int lo, int hi, double& sum, double& plain) {
  constexpr int EPL = Pack<DT>::EPL, U = 16 / EPL, STEP = 64 * EPL;   // 16 entries in hand
  const int lane = __lane_id();
  sum = plain = 0.0;
  const int i0 = w.rej ? __ffsll(static_cast<long long>(w.rej)) - 1 : 0;
  const double z0 = w.rej ? readlane_f64(z, i0) : 0.0;
  for (int v0 = lo; v0 + EPL <= hi; v0 += U * STEP) {
    u32x4 p[U], q[U];
    double r[U][EPL];
    bool in[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int v = v0 + k * STEP + lane * EPL;
      in[k] = v + EPL <= hi;
      p[k] = load_pack<DT>(w.p, in[k] ? v : lo);
      // the first rejected draft's row together with it (where there is none: the same row once more)
      if constexpr (DRAFT) q[k] = load_pack<DT>(w.rej ? w.draft : w.p, (w.rej ? i0 * w.d_row : 0) + (in[k] ? v : lo));
    }
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const float t = element<DT>(p[k], e);
        r[k][e] = in[k] && t > 0.f ? t : 0.f;
        if (PLAIN) plain += r[k][e];
        if constexpr (DRAFT) r[k][e] = fmax(r[k][e] - z0 * static_cast<double>(element<DT>(q[k], e)), 0.0);
      }
    for (u64 rest = DRAFT ? w.rej & (w.rej - 1) : w.rej; rest; rest &= rest - 1) {
      const int i = __ffsll(static_cast<long long>(rest)) - 1;
      if constexpr (DRAFT) {
        const double zi = readlane_f64(z, i);
#pragma unroll
        for (int k = 0; k < U; ++k) {
          const u32x4 y = load_pack<DT>(w.draft, i * w.d_row + (in[k] ? v0 + k * STEP + lane * EPL : lo));
#pragma unroll
          for (int e = 0; e < EPL; ++e) r[k][e] = fmax(r[k][e] - zi * static_cast<double>(element<DT>(y, e)), 0.0);
        }
      } else {
        const int xi = __builtin_amdgcn_readlane(x, i);
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
          for (int e = 0; e < EPL; ++e) r[k][e] = v0 + k * STEP + lane * EPL + e == xi ? 0.0 : r[k][e];
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int e = 0; e < EPL; ++e) sum += r[k][e];
  }
  // a last pack that the range's end cuts
  const int tail = lo + max(hi - lo, 0) / EPL * EPL + lane;
  if (__any(tail < hi)) {
    const double r = weight<DT, DRAFT>(w, z, x, tail < hi ? tail : lo);
    const float t = ld1<DT>(w.p, tail < hi ? tail : lo);
    sum += tail < hi ? r : 0.0;
    if (PLAIN) plain += tail < hi && t > 0.f ? t : 0.0;
  }
}

// ws of a sequence: the walk's end, then the sums of the row's pieces (R, row), one a wave of each slice
struct WalkEnd {
  u64 rej;
  int cur, pad;
  double z[kTreePlaces];
};
__device__ __forceinline__ WalkEnd* walk_end(const TreeVerifyArgs& a, int b) { return static_cast<WalkEnd*>(a.ws) + b; }
__device__ __forceinline__ double* pieces_of(const TreeVerifyArgs& a, int b) {
  return reinterpret_cast<double*>(static_cast<WalkEnd*>(a.ws) + a.B) + static_cast<int64_t>(b) * a.slices * kWaves * 2;
}
// entries of piece j: slice j / kWaves, wave j % kWaves of it
__device__ __forceinline__ void piece(const TreeVerifyArgs& a, int j, int& lo, int& hi) {
  const int s0 = j / kWaves * a.per, s1 = min(a.V, s0 + a.per), len = (a.per + kWaves - 1) / kWaves;
  lo = min(s1, s0 + j % kWaves * len);
  hi = min(s1, lo + len);
}

// Running sum over the workgroup's threads, and the whole (the same bits in every thread).
__device__ __forceinline__ double block_scan(double x, double* lds, double& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double s = wave_scan(x);
  if (lane == 63) lds[wave] = s;
  __syncthreads();
  double before = 0.0;
  total = 0.0;
#pragma unroll
  for (int k = 0; k < kWaves; ++k) {
    before += k < wave ? lds[k] : 0.0;
    total += lds[k];
  }
  __syncthreads();
  return s + before;
}
// The first thread that says `hit`, else the last that says `has` (one does), in all threads.
__device__ __forceinline__ int block_pick(bool hit, bool has, int* lds) {
  if (threadIdx.x == 0) {
    lds[0] = kThreads;
    lds[1] = -1;
  }
  __syncthreads();
  const u64 h = __ballot(hit), l = __ballot(has);
  const int first = threadIdx.x & ~63;
  if ((threadIdx.x & 63) == 0) {
    if (h) atomicMin(&lds[0], first + __ffsll(static_cast<long long>(h)) - 1);
    if (l) atomicMax(&lds[1], first + 63 - __clzll(static_cast<long long>(l)));
  }
  __syncthreads();
  const int r = lds[0] < kThreads ? lds[0] : lds[1];
  __syncthreads();
  return r;
}

// The lowest v whose running sum of R passes u times the sum: the piece of the row, then
// the thread whose few entries of it, then the entry.  sums: of the pieces, R and the row.
template <int DT, bool DRAFT>
__device__ __forceinline__ void pick(const TreeVerifyArgs& a, int b, const double* sums, const Weights& given, double z, int x, double u) {
  __shared__ double lds[kWaves];
  __shared__ int which[2];
  const int n = a.slices * kWaves;       // at most as many as threads
  Weights w = given;
  const int tid = threadIdx.x;
  double own = tid < n ? sums[2 * tid] : 0.0, total;
  double scan = block_scan(own, lds, total);
  if (!(total > 0.0)) {                  // nothing left: the row as it was
    w.rej = 0;
    own = tid < n ? sums[2 * tid + 1] : 0.0;
    scan = block_scan(own, lds, total);
    if (!(total > 0.0)) {
      if (tid == 0) a.next[b] = -1;
      return;
    }
  }
  // past every sum (u not below 1): the last that has a weight
  const double t = u * total;
  const int j = block_pick(own > 0.0 && scan > t, own > 0.0, which);
  if (tid == j) lds[0] = scan - own;
  __syncthreads();
  const double before = lds[0];
  __syncthreads();
  int lo, hi;
  piece(a, j, lo, hi);
  const int len = (hi - lo + kThreads - 1) / kThreads, v0 = lo + tid * len;
  double c = 0.0;
  for (int e = 0; e < len; ++e) {
    const double r = weight<DT, DRAFT>(w, z, x, v0 + e < hi ? v0 + e : lo);
    c += v0 + e < hi ? r : 0.0;
  }
  const double cs = block_scan(c, lds, total);
  const int at = block_pick(c > 0.0 && before + cs > t, c > 0.0, which);
  // no entry has a weight only if the piece's sum has none
  if (at < 0) {
    if (tid == 0) a.next[b] = lo;
    return;
  }
  if ((tid & ~63) == (at & ~63)) {       // the wave of that thread: weight() reads over its lanes
    double acc = before + cs - c;
    int found = -1;
    bool done = false;
    for (int e = 0; e < len; ++e) {
      const double r = weight<DT, DRAFT>(w, z, x, v0 + e < hi ? v0 + e : lo);
      if (v0 + e < hi && r > 0.0 && !done) {
        found = v0 + e;
        acc += r;
        done = acc > t;
      }
    }
    if (tid == at) a.next[b] = found;
  }
}

// A workgroup a (slice, sequence).  Every wave walks the tree (the same numbers, the
// same decisions); where a rejected child has a sibling to ask, the workgroup sums
// the row that is left.  Then the waves sum their pieces of the slice.
template <int DT, bool DRAFT>
__global__ __launch_bounds__(kThreads) void kda_tree_sample_kernel(TreeVerifyArgs a) {
  __shared__ double red[2][kWaves];
  __shared__ double sums[2 * kWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int s = blockIdx.y, b = blockIdx.z * gridDim.x + blockIdx.x, N = a.N, mine = min(lane, N - 1);
  if (b >= a.B) return;
  const int parent = a.parents[static_cast<int64_t>(b) * N + mine];
  const int64_t x64 = a.tokens[static_cast<int64_t>(b) * N + mine];
  const double u = a.uniforms[static_cast<int64_t>(b) * (N + 1) + mine], u_next = a.uniforms[static_cast<int64_t>(b) * (N + 1) + N];
  const bool live = tree_paths(parent, N) != 0, real = live && x64 >= 0 && x64 < a.V;
  const int x = real ? static_cast<int>(x64) : -1;
  constexpr int ES = DT == 0 ? 4 : 2;
  const char* target = static_cast<const char*>(a.target) + b * a.t_b * ES;
  Weights w{target, DRAFT ? static_cast<const char*>(a.draft) + b * a.d_b * ES : nullptr, a.d_row, 0};
  double r = real ? ld1<DT>(target, (parent + 1) * a.t_row + x) : 0.0;
  const double q = !DRAFT ? 1.0 : real ? ld1<DT>(w.draft, lane * a.d_row + x) : 0.0;

  int cur = -1, count = 0, turn = 0;
  double Z = 1.0, z = 0.0;
  u64 kids = __ballot(live && parent == -1);
  while (kids) {
    const int i = __ffsll(static_cast<long long>(kids)) - 1;
    kids &= kids - 1;
    const double ri = readlane_f64(r, i);
    if (readlane_f64(u, i) * readlane_f64(q, i) * Z < ri) {
      cur = i;
      ++count;
      Z = 1.0;
      w.p = target + (i + 1) * a.t_row * ES;
      w.rej = 0;
      kids = __ballot(live && parent == i);
      continue;
    }
    if (lane == i) z = Z;
    w.rej |= u64{1} << i;
    if (!kids) break;
    if constexpr (DRAFT) {
      // A wave's entries in four parts, which the slices take in turns: what one fetches another finds in
      // its L2 (cold 47.2 us for 49.6).  The parts' sums are added in one order, so all see one Z.
      constexpr int ROUND = 1024;
      const int len = ((a.V + kWaves - 1) / kWaves + 63) & ~63, cut = len < 4 * ROUND ? len : (len / 4 + ROUND - 1) / ROUND * ROUND;
      const int end = min(a.V, (wave + 1) * len);
      double quarter[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 1
      for (int t = 0; t < 4; ++t) {
        const int k = (t + s) & 3, from = wave * len + k * cut;
        if (from >= end) continue;
        double part, plain;
        sum_range<DT, DRAFT, false>(w, z, x, from, min(end, from + cut), part, plain);
#pragma unroll
        for (int y = 0; y < 4; ++y) quarter[y] = y == k ? part : quarter[y];
      }
      double sum = wave_sum((quarter[0] + quarter[1]) + (quarter[2] + quarter[3]));
      if (lane == 0) red[turn][wave] = sum;
      const double qx = real ? ld1<DT>(w.draft, i * a.d_row + x) : 0.0;
      if ((kids >> lane) & 1) r = fmax(r - Z * qx, 0.0);   // of the children still to ask
      lds_barrier();
      Z = 0.0;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) Z += red[turn][k];
      turn ^= 1;
    } else {
      Z = fmax(Z - (ri > 0.0 ? ri : 0.0), 0.0);
      if (parent == cur && x == __builtin_amdgcn_readlane(x, i)) r = 0.0;
    }
  }

  int lo, hi;
  piece(a, s * kWaves + wave, lo, hi);
  double sum, plain;
  sum_range<DT, DRAFT, true>(w, z, x, lo, hi, sum, plain);
  sum = wave_sum(sum);
  plain = wave_sum(plain);
  double* out = a.slices == 1 ? sums : pieces_of(a, b) + 2 * s * kWaves;
  if (lane == 0) {
    out[2 * wave] = sum;
    out[2 * wave + 1] = plain;
  }
  if (s == 0 && wave == 0) {
    if (lane == 0) {
      a.last[b] = cur;
      a.accepted[b] = count;
    }
    if (a.slices > 1) {
      WalkEnd* e = walk_end(a, b);
      e->z[lane] = z;
      if (lane == 0) {
        e->rej = w.rej;
        e->cur = cur;
      }
    }
  }
  if (a.slices == 1) {
    __syncthreads();
    pick<DT, DRAFT>(a, b, sums, w, z, x, u_next);
  }
}

// The next token of a sequence whose row was summed in slices.
template <int DT, bool DRAFT>
__global__ __launch_bounds__(kThreads) void kda_tree_pick_kernel(TreeVerifyArgs a) {
  constexpr int ES = DT == 0 ? 4 : 2;
  const int b = blockIdx.x, lane = threadIdx.x & 63;
  const WalkEnd* e = walk_end(a, b);
  const int64_t x64 = a.tokens[static_cast<int64_t>(b) * a.N + min(lane, a.N - 1)];
  const Weights w{static_cast<const char*>(a.target) + (b * a.t_b + (__builtin_amdgcn_readfirstlane(e->cur) + 1) * a.t_row) * ES,
                  DRAFT ? static_cast<const char*>(a.draft) + b * a.d_b * ES : nullptr, a.d_row, uniform_u64(e->rej)};
  const int x = x64 >= 0 && x64 < a.V ? static_cast<int>(x64) : -1;
  pick<DT, DRAFT>(a, b, pieces_of(a, b), w, e->z[lane], x, a.uniforms[static_cast<int64_t>(b) * (a.N + 1) + a.N]);
}

// ------------------------------------------------------------------ greedy
// A value as a whole number in its order; larger and then lower index first.
__device__ __forceinline__ u64 best_key(float x, int v) {
  unsigned o = __float_as_uint(x + 0.f);   // -0 is 0
  o = o & 0x80000000u ? ~o : o | 0x80000000u;
  return static_cast<u64>(o) << 32 | static_cast<unsigned>(~v);
}
__device__ __forceinline__ u64 wave_max(u64 x) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) {
    const u64 y = shfl_u64(x, __lane_id() ^ s);
    x = y > x ? y : x;
  }
  return x;
}
// Key of the largest entry of [lo, hi) of a row, in all lanes; 0: all NaN.
template <int DT>
__device__ __forceinline__ u64 best_of(const void* row, int lo, int hi) {
  constexpr int EPL = Pack<DT>::EPL, U = 4, STEP = 64 * EPL;
  const int lane = __lane_id();
  float top = -INFINITY;
  int at = -1;
  auto see = [&](float x, int v) {
    if (x > top || (at < 0 && x == top)) {   // a lane sees its entries in rising order
      top = x;
      at = v;
    }
  };
  for (int v0 = lo; v0 + EPL <= hi; v0 += U * STEP) {
    u32x4 t[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int v = v0 + k * STEP + lane * EPL;
      t[k] = load_pack<DT>(row, v + EPL <= hi ? v : lo);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int v = v0 + k * STEP + lane * EPL;
      if (v + EPL <= hi)
#pragma unroll
        for (int e = 0; e < EPL; ++e) see(element<DT>(t[k], e), v + e);
    }
  }
  const int tail = lo + (hi - lo) / EPL * EPL + lane;
  if (hi > lo && tail < hi) see(ld1<DT>(row, tail), tail);
  return wave_max(at < 0 ? 0 : best_key(top, at));
}

// The largest entry of a slice of a row: a workgroup each, of every row that a walk can reach (which
// one it does is known only after the rows before it).  Bound by their bytes where
// there are many, 64 sequences of 16 places and 128000 bf16 61 us for 279 MB, of which a walk over
// three rows needs 49; 16 of 8 places and 50021 bf16 7, and 3 of the walk's launch.
template <int DT>
__global__ __launch_bounds__(256) void kda_tree_best_kernel(TreeVerifyArgs a) {
  constexpr int ES = DT == 0 ? 4 : 2;
  __shared__ u64 red[4];
  const int s = blockIdx.x % a.slices, row = blockIdx.x / a.slices, b = row / (a.N + 1), i = row - b * (a.N + 1);
  if (i > 0) {
    const int parent = a.parents[static_cast<int64_t>(b) * a.N + i - 1];
    if (parent < -1 || parent >= i - 1) return;    // no draft here: no walk reads this row
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), len = (a.per + 3) / 4;
  const int s0 = s * a.per, s1 = min(a.V, s0 + a.per), lo = min(s1, s0 + wave * len), hi = min(s1, lo + len);
  const u64 k = best_of<DT>(static_cast<const char*>(a.target) + (b * a.t_b + i * a.t_row) * ES, lo, hi);
  if ((threadIdx.x & 63) == 0) red[wave] = k;
  __syncthreads();
  if (threadIdx.x == 0) {
    u64 m = red[0];
    for (int y = 1; y < 4; ++y) m = red[y] > m ? red[y] : m;
    static_cast<u64*>(a.ws)[static_cast<int64_t>(row) * a.slices + s] = m;
  }
}
__device__ __forceinline__ int token_of(u64 key) { return key ? static_cast<int>(~static_cast<unsigned>(key)) : 0; }
__global__ __launch_bounds__(64) void kda_tree_greedy_kernel(TreeVerifyArgs a) {
  const int b = blockIdx.x, lane = threadIdx.x, N = a.N, mine = min(lane, N - 1);
  const int parent = a.parents[static_cast<int64_t>(b) * N + mine];
  const int64_t x = a.tokens[static_cast<int64_t>(b) * N + mine];
  const u64* keys = static_cast<const u64*>(a.ws) + static_cast<int64_t>(b) * (N + 1) * a.slices;
  const bool live = tree_paths(parent, N) != 0;
  u64 own = 0, root = 0;
  for (int s = lane; s < a.slices; s += 64) root = keys[s] > root ? keys[s] : root;
  if (live)
    for (int s = 0; s < a.slices; ++s) {
      const u64 k = keys[static_cast<int64_t>(mine + 1) * a.slices + s];
      own = k > own ? k : own;
    }
  const int best = token_of(own);
  int cur = -1, count = 0, word = token_of(wave_max(root));
  for (;;) {
    const u64 kids = __ballot(live && parent == cur && x == word);
    if (!kids) break;
    cur = __ffsll(static_cast<long long>(kids)) - 1;
    ++count;
    word = __builtin_amdgcn_readlane(best, cur);
  }
  if (lane == 0) {
    a.last[b] = cur;
    a.accepted[b] = count;
    a.next[b] = word;
  }
}

template <int DT>
hipError_t verify(const TreeVerifyArgs& a, hipStream_t s) {
  if (!a.uniforms) {
    kda_tree_best_kernel<DT><<<dim3(static_cast<unsigned>(a.B) * (a.N + 1) * a.slices), dim3(256), 0, s>>>(a);
    kda_tree_greedy_kernel<<<dim3(a.B), dim3(64), 0, s>>>(a);
    return hipGetLastError();
  }
  // A sequence's slices eight workgroups apart, on one XCD, whose L2 then serves the rows that
  // all of them sum: 64 sequences of 128000 fp32 entries, warm, 30.1 us for 32.9; fewer than
  // eight would leave XCDs idle.
  const unsigned wide = a.slices > 1 ? (a.B >= 8 ? 8 : 1) : a.B;
  const dim3 grid(wide, a.slices, (a.B + wide - 1) / wide), block(kThreads);
  if (a.draft) kda_tree_sample_kernel<DT, true><<<grid, block, 0, s>>>(a);
  else kda_tree_sample_kernel<DT, false><<<grid, block, 0, s>>>(a);
  if (a.slices > 1) {
    if (a.draft) kda_tree_pick_kernel<DT, true><<<dim3(a.B), block, 0, s>>>(a);
    else kda_tree_pick_kernel<DT, false><<<dim3(a.B), block, 0, s>>>(a);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_tree_verify(const TreeVerifyArgs& a, int dt, hipStream_t s) {
  return dt == 0 ? verify<0>(a, s) : dt == 1 ? verify<1>(a, s) : verify<2>(a, s);
}

}  // namespace kda
