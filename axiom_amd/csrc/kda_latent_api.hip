// C ABI of the latent attention: argument validation, workspace layout, dispatch.
#include "latent_mi355x.h"

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <initializer_list>

#include "kda_internal.h"

namespace {

int fail(int code, const char* fmt, ...) {
  char msg[400];
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  return kda::api_fail(code, msg);
}
int launched(hipError_t e, const char* what) {
  return e == hipSuccess ? KDA_OK : fail(KDA_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}
size_t align_up(size_t x) { return (x + 255) / 256 * 256; }
bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
size_t elem(int dtype) { return dtype == KDA_DTYPE_F32 ? 4 : 2; }
bool dtype_ok(int dtype) { return dtype == KDA_DTYPE_F32 || dtype == KDA_DTYPE_BF16 || dtype == KDA_DTYPE_F16; }

// A tile's rows are addressed with 32-bit offsets from its first row: 64 rows at most.
constexpr int64_t kMaxRowBytes = int64_t{1} << 25;
constexpr int64_t kMaxBlocks = int64_t{1} << 23;   // 256 threads each

int check_attn(const void* q, const void* kv, const void* kr, const int64_t* st, const int32_t* cu_q, const int32_t* cu_k,
               int32_t n_seqs, int B, int Tq, int Tk, int H, int dn, int dr, float scale, int dtype) {
  if (!dtype_ok(dtype)) return fail(KDA_ERR_INVALID_ARGUMENT, "dtype=%d must be F32, BF16 or F16", dtype);
  if (B < 0 || Tq < 0 || Tk < 0 || H < 1) return fail(KDA_ERR_INVALID_ARGUMENT, "sizes B=%d Tq=%d Tk=%d H=%d out of range", B, Tq, Tk, H);
  if ((dn != 64 && dn != 128) || (dr != 32 && dr != 64))
    return fail(KDA_ERR_UNSUPPORTED, "head dims dn=%d, dr=%d unsupported (dn in {64, 128}, dr in {32, 64})", dn, dr);
  if (!(scale > 0.f) || !std::isfinite(scale)) return fail(KDA_ERR_INVALID_ARGUMENT, "scale must be positive and finite");
  if ((cu_q == nullptr) != (cu_k == nullptr)) return fail(KDA_ERR_INVALID_ARGUMENT, "cu_q and cu_k go together");
  if (cu_q && (B != 1 || n_seqs < 1)) return fail(KDA_ERR_INVALID_ARGUMENT, "packed sequences need B == 1 and n_seqs >= 1");
  if (static_cast<int64_t>(B) * H > 65535) return fail(KDA_ERR_UNSUPPORTED, "B * H = %lld over 65535", static_cast<long long>(B) * H);
  const int64_t blocks = (static_cast<int64_t>(Tq > Tk ? Tq : Tk) / 128 + 1 + (cu_q ? n_seqs : 0)) * B * H;
  if (blocks > kMaxBlocks) return fail(KDA_ERR_UNSUPPORTED, "%lld blocks of 128 rows over %lld", static_cast<long long>(blocks),
                                       static_cast<long long>(kMaxBlocks));
  if (!st) return fail(KDA_ERR_INVALID_ARGUMENT, "null strides");
  if (static_cast<int64_t>(B) * Tq > 0 && !q) return fail(KDA_ERR_INVALID_ARGUMENT, "null q");
  if (static_cast<int64_t>(B) * Tk > 0 && (!kv || !kr)) return fail(KDA_ERR_INVALID_ARGUMENT, "null kv or k_rope");
  for (const void* p : {q, kv, kr})
    if (!aligned(p, 16)) return fail(KDA_ERR_INVALID_ARGUMENT, "q, kv and k_rope must be aligned to 16 bytes");
  const int64_t es = static_cast<int64_t>(elem(dtype));
  for (int i = 0; i < 8; ++i)
    if (st[i] < 0 || st[i] * es % 16 != 0)
      return fail(KDA_ERR_INVALID_ARGUMENT, "strides must be non-negative multiples of 16 bytes (stride %d is %lld elements)", i,
                  static_cast<long long>(st[i]));
  if (st[1] * es >= kMaxRowBytes || st[4] * es >= kMaxRowBytes || st[7] * es >= kMaxRowBytes)
    return fail(KDA_ERR_UNSUPPORTED, "token strides of 32 MiB or more are unsupported");
  return KDA_OK;
}

bool sizes_ok(int B, int Tq, int Tk, int H, int dn, int dr, int n_seqs, int dtype) {
  return B >= 0 && Tq >= 0 && Tk >= 0 && H >= 1 && (dn == 64 || dn == 128) && (dr == 32 || dr == 64) && n_seqs >= 0 && dtype_ok(dtype);
}

kda::LatentArgs attn_args(const void* q, const void* kv, const void* kr, const int64_t* st, const int32_t* cu_q,
                          const int32_t* cu_k, int32_t n_seqs, int B, int Tq, int Tk, int H, int causal, float scale) {
  kda::LatentArgs a{};
  a.q = q; a.kv = kv; a.kr = kr;
  a.cu_q = cu_q; a.cu_k = cu_k; a.n_seqs = cu_q ? n_seqs : 0;
  a.B = B; a.Tq = Tq; a.Tk = Tk; a.H = H;
  a.q_b = st[0]; a.q_t = st[1]; a.q_h = st[2];
  a.kv_b = st[3]; a.kv_t = st[4]; a.kv_h = st[5];
  a.kr_b = st[6]; a.kr_t = st[7];
  a.causal = causal != 0;
  a.scale = scale;
  return a;
}

// Shares of a block of 128 rows along the other axis.  A launch of fewer blocks
// than the chip runs at once leaves CUs idle while each block walks its whole
// row of tiles, so the walks are cut into shares of `len` tiles (up to 16 a
// block, 128 rows each at least), as short as kSlots workgroups allow; a join
// adds their fp32 parts.  Equal lengths, not equal numbers: a causal call's walks
// differ, and its longest share is what it waits for (fp32 B1 H8 T1024
// forward and backward 256 us with equal numbers, 195 with these; bf16 1 x 1000 of
// d 64 the five kernels 72 us, 65).  `live`:
// the shares of a head's blocks, one a workgroup of the grid (a grid of blocks by
// the most shares, its empty workgroups leaving at once, put two of the others on
// some CUs: 1.3 times as long).  Not where the longest walk falls by less than a
// quarter.  Packed lengths are on the device: there `parts` equal shares of each
// block (len 0).
// kSlots: one workgroup a CU, and no shares past as many blocks.  Against 512 (bf16,
// forward / backward): T = 1000 H8 d 64, 64 blocks, 13.9 / 38.5 us and 14.4 / 48.7; T =
// 2048 H8, 128 blocks, 31.1 / 95.0 and 34.6 / 108; but T = 2560 H12, 240 blocks, 58 / 212
// and 48 / 176, and T = 4096 H8, 256 blocks, 89 / 322 and 67 / 241: from some 200
// causal blocks up the longest walk is twice the mean, and 256 workgroups leave
// nothing to even it out with.  At 512 blocks neither shares any.
constexpr int kSlots = 256;
struct Shares { int len, parts, live; };
// blocks of 128 rows of one head; packed: every sequence ends in at most one partial block
int64_t blocks_of(int64_t T, int n_seqs) { return n_seqs > 0 ? T / 128 + n_seqs : (T + 127) / 128; }
// q_side: blocks of queries that walk keys, else keys that walk queries
Shares shares_of(bool q_side, int64_t Tq, int64_t Tk, int64_t heads, int n_seqs, bool causal, int dtype) {
  const int64_t T = q_side ? Tq : Tk, other = q_side ? Tk : Tq, blocks = blocks_of(T, n_seqs);
  const int64_t most = std::min<int64_t>(16, (other + 127) / 128);
  if (blocks <= 0 || blocks * heads > kSlots || most <= 1) return {0, 1, 0};
  if (n_seqs > 0) return {0, static_cast<int>(std::max<int64_t>(1, std::min(kSlots / (blocks * heads), most))), 0};
  const int64_t tile = dtype == KDA_DTYPE_F32 ? 32 : 64, all = (other + tile - 1) / tile;
  auto walk = [&](int64_t i) {
    if (!causal) return all;
    if (q_side) return std::max<int64_t>(0, std::min(Tk - 1, std::min(128 * i + 127, Tq - 1) + Tk - Tq) + tile) / tile;
    return std::max<int64_t>(0, all - std::max<int64_t>(0, 128 * i + Tq - Tk) / tile);
  };
  const int64_t longest = walk(q_side ? blocks - 1 : 0);
  auto live = [&](int64_t len) {
    int64_t n = 0;
    for (int64_t i = 0; i < blocks; ++i) n += std::max<int64_t>(1, (walk(i) + len - 1) / len);
    return n;
  };
  int64_t lo = std::max<int64_t>(128 / tile, (longest + most - 1) / most), hi = longest;
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (live(mid) * heads <= kSlots) hi = mid;
    else lo = mid + 1;
  }
  if (4 * lo > 3 * longest) return {0, 1, 0};
  return {static_cast<int>(lo), static_cast<int>((longest + lo - 1) / lo), static_cast<int>(live(lo))};
}

struct FwdLayout { Shares q; size_t ml, total; };
FwdLayout fwd_layout(int B, int Tq, int Tk, int H, int dn, int n_seqs, bool causal, int dtype) {
  FwdLayout L{};
  const int64_t bh = static_cast<int64_t>(B) * H;
  L.q = shares_of(true, Tq, Tk, bh, n_seqs, causal, dtype);
  const size_t rows = L.q.parts > 1 ? static_cast<size_t>(L.q.parts) * bh * Tq : 0;
  L.ml = align_up(rows * dn * 4);
  L.total = L.ml + align_up(rows * 8);
  return L;
}
struct BwdLayout { Shares q, k; size_t D, dkr, part, part_k, total; };
BwdLayout bwd_layout(int B, int Tq, int Tk, int H, int dn, int dr, int n_seqs, bool causal, int dtype) {
  BwdLayout L{};
  const size_t bh = static_cast<size_t>(B) * H;
  L.q = shares_of(true, Tq, Tk, static_cast<int64_t>(bh), n_seqs, causal, dtype);
  L.k = shares_of(false, Tq, Tk, static_cast<int64_t>(bh), n_seqs, causal, dtype);
  L.D = 0;
  // after D, room for 4 bytes a query block that no kernel uses: the size of a
  // workspace stays what it was while one did
  L.dkr = align_up(bh * Tq * 4) + align_up(bh * blocks_of(Tq, n_seqs) * 4);
  L.part = L.dkr + align_up(L.k.parts * bh * Tk * dr * 4);
  L.part_k = L.part + align_up(L.q.parts > 1 ? L.q.parts * bh * Tq * (dn + dr) * 4 : 0);
  L.total = L.part_k + align_up(L.k.parts > 1 ? L.k.parts * bh * Tk * 2 * dn * 4 : 0) + 256;
  return L;
}

// Decode: query rows of a workgroup (16, or 64 where there are more than 16;
// fp32 16, whose operands take twice the registers and LDS), the row groups
// of a sequence, and the workgroups along the cache: one a CU (its buffers take
// the LDS), and no more than there can be runs of `least` tiles.  Sequences whose
// table holds at most kWholeTokens tokens get a workgroup each instead and no join
// launch: R512 bf16, 16 rows, tables of 128 tokens 11.8 us for one sequence and 14.0
// for 256, in runs 12.6 and 20.4; of 192 tokens 13.8 and 16.5, in runs 12.7 and 23.0, so
// from there on it is the number of sequences that decides, and runs are taken.
// pad, the places of a sequence beside its tiles (16 rows; 64 sequences of 1 to
// 8192 tokens and 256 of 1 to 1024): 0 62 and 65 us, 4 40 and 33, 8 34 and 30, 16 34 and
// 34; 64 rows: 0 83 and 70, 2 55 and 54, 4 46 and 49, 8 46 and 50.
// least: 2 and 1 are alike but for 64 rows of one sequence of 4096 tokens (22 and
// 28 us); 4 takes 17.1 for 19.4 with 16 rows there, and 14.2 for 13.4 at 512 tokens.
constexpr int kCUs = 256;
constexpr int kWholeTokens = 128;
struct DecodePlan { int rows, groups, wgs, whole, least, pad; size_t part_ml, part_o, total; };
bool decode_plan(int B, int Tq, int H, int R, int page_size, int max_pages, int dtype, DecodePlan* P) {
  const int64_t rows = static_cast<int64_t>(Tq) * H, cap = static_cast<int64_t>(page_size) * max_pages;
  P->rows = rows <= 16 || dtype == KDA_DTYPE_F32 ? 16 : 64;
  P->least = 2;
  P->pad = P->rows == 64 ? 4 : 8;
  const int64_t kt = kda::latent_decode_tile(P->rows), tiles = ((cap + kt - 1) / kt + P->pad) * B;
  if (rows > (1 << 20) || cap >= (int64_t{1} << 31) || tiles >= (int64_t{1} << 30)) return false;
  P->groups = static_cast<int>((rows + P->rows - 1) / P->rows);
  P->whole = cap <= kWholeTokens;
  const int64_t wgs = kCUs / P->groups > 8 ? kCUs / P->groups / 8 * 8 : 8, runs = (tiles + P->least - 1) / P->least;
  P->wgs = P->whole ? (B > 0 ? B : 1) : static_cast<int>(wgs < runs ? wgs : runs);
  const size_t slots = P->whole ? 0 : 2 * static_cast<size_t>(P->wgs) * P->groups * P->rows;
  P->part_ml = align_up(4 * (static_cast<size_t>(B) + 1));
  P->part_o = P->part_ml + align_up(slots * 8);
  P->total = P->part_o + align_up(slots * R * 4);
  return true;
}
bool pow2(int x) { return x > 0 && (x & (x - 1)) == 0; }

}  // namespace

extern "C" {

int kda_latent_attn_fwd(hipStream_t stream, const void* q, const void* kv, const void* k_rope, const int64_t* strides,
                        const int32_t* cu_q, const int32_t* cu_k, int32_t n_seqs, void* o, float* lse, int B, int Tq, int Tk,
                        int H, int dn, int dr, int causal, float scale, int dtype, void* workspace, size_t workspace_bytes) {
  if (const int rc = check_attn(q, kv, k_rope, strides, cu_q, cu_k, n_seqs, B, Tq, Tk, H, dn, dr, scale, dtype)) return rc;
  if (static_cast<int64_t>(B) * Tq == 0) return KDA_OK;
  if (!o || !lse) return fail(KDA_ERR_INVALID_ARGUMENT, "null o or lse");
  if (!aligned(o, 16)) return fail(KDA_ERR_INVALID_ARGUMENT, "o must be aligned to 16 bytes");
  const FwdLayout L = fwd_layout(B, Tq, Tk, H, dn, cu_q ? n_seqs : 0, causal != 0, dtype);
  if (L.total > 0 && (!workspace || workspace_bytes < L.total))
    return fail(KDA_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : size_t{0}, L.total);
  if (!aligned(workspace, 16)) return fail(KDA_ERR_INVALID_ARGUMENT, "workspace must be aligned to 16 bytes");
  kda::LatentArgs a = attn_args(q, kv, k_rope, strides, cu_q, cu_k, n_seqs, B, Tq, Tk, H, causal, scale);
  a.o = o;
  a.lse = lse;
  a.splits = L.q.parts; a.share = L.q.len; a.live = L.q.live;
  a.part = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + L.ml);
  return launched(kda::launch_latent_fwd(a, dn, dr, dtype, stream), "kda_latent_attn_fwd");
}

size_t kda_latent_attn_fwd_workspace(int B, int Tq, int Tk, int H, int dn, int dr, int32_t n_seqs, int dtype) {
  if (!sizes_ok(B, Tq, Tk, H, dn, dr, n_seqs, dtype)) return 0;
  return std::max(fwd_layout(B, Tq, Tk, H, dn, n_seqs, false, dtype).total, fwd_layout(B, Tq, Tk, H, dn, n_seqs, true, dtype).total);
}

size_t kda_latent_attn_bwd_workspace(int B, int Tq, int Tk, int H, int dn, int dr, int32_t n_seqs, int dtype) {
  if (!sizes_ok(B, Tq, Tk, H, dn, dr, n_seqs, dtype)) return 0;
  return std::max(bwd_layout(B, Tq, Tk, H, dn, dr, n_seqs, false, dtype).total,
                  bwd_layout(B, Tq, Tk, H, dn, dr, n_seqs, true, dtype).total);
}

int kda_latent_attn_bwd(hipStream_t stream, const void* q, const void* kv, const void* k_rope, const int64_t* strides,
                        const int32_t* cu_q, const int32_t* cu_k, int32_t n_seqs, const void* o, const float* lse,
                        const void* d_o, void* dq, void* dkv, void* dk_rope, int B, int Tq, int Tk, int H, int dn, int dr,
                        int causal, float scale, int dtype, void* workspace, size_t workspace_bytes) {
  if (const int rc = check_attn(q, kv, k_rope, strides, cu_q, cu_k, n_seqs, B, Tq, Tk, H, dn, dr, scale, dtype)) return rc;
  if (B == 0) return KDA_OK;
  if (Tq > 0 && (!o || !lse || !d_o || !dq)) return fail(KDA_ERR_INVALID_ARGUMENT, "null o, lse, d_o or dq");
  if (Tk > 0 && (!dkv || !dk_rope)) return fail(KDA_ERR_INVALID_ARGUMENT, "null dkv or dk_rope");
  for (const void* p : {o, d_o, static_cast<const void*>(dq), static_cast<const void*>(dkv), static_cast<const void*>(dk_rope)})
    if (!aligned(p, 16)) return fail(KDA_ERR_INVALID_ARGUMENT, "o, d_o, dq, dkv and dk_rope must be aligned to 16 bytes");
  if (static_cast<int64_t>(H) * dn * elem(dtype) >= kMaxRowBytes) return fail(KDA_ERR_UNSUPPORTED, "H * dn too large");
  const BwdLayout L = bwd_layout(B, Tq, Tk, H, dn, dr, cu_q ? n_seqs : 0, causal != 0, dtype);
  if (!workspace || workspace_bytes < L.total)
    return fail(KDA_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : size_t{0}, L.total);
  if (!aligned(workspace, 16)) return fail(KDA_ERR_INVALID_ARGUMENT, "workspace must be aligned to 16 bytes");
  kda::LatentArgs a = attn_args(q, kv, k_rope, strides, cu_q, cu_k, n_seqs, B, Tq, Tk, H, causal, scale);
  char* ws = static_cast<char*>(workspace);
  a.o_in = o; a.lse_in = lse; a.dout = d_o;
  a.D = reinterpret_cast<float*>(ws + L.D);
  a.dkr_part = reinterpret_cast<float*>(ws + L.dkr);
  a.part = reinterpret_cast<float*>(ws + L.part);
  a.part_k = reinterpret_cast<float*>(ws + L.part_k);
  a.splits = L.q.parts; a.share = L.q.len; a.live = L.q.live;
  a.splits_k = L.k.parts; a.share_k = L.k.len; a.live_k = L.k.live;
  a.dq = dq; a.dkv = dkv; a.dkr = dk_rope;
  return launched(kda::launch_latent_bwd(a, dn, dr, dtype, stream), "kda_latent_attn_bwd");
}

int kda_latent_append(hipStream_t stream, const void* rows, int64_t rows_stride, const int64_t* positions, const int64_t* slots,
                      const float* cos_sin, int64_t n_positions, const float* norm_weight, float eps, void* cache,
                      int64_t n_slots, const void* q, int64_t q_stride_t, int64_t q_stride_h, void* q_out, int64_t qo_stride_t,
                      int64_t qo_stride_h, int N, int H, int R, int dr, int interleaved, int dtype) {
  if (!dtype_ok(dtype)) return fail(KDA_ERR_INVALID_ARGUMENT, "dtype=%d must be F32, BF16 or F16", dtype);
  if ((R != 256 && R != 512) || (dr != 32 && dr != 64))
    return fail(KDA_ERR_UNSUPPORTED, "R=%d, dr=%d unsupported (R in {256, 512}, dr in {32, 64})", R, dr);
  if (N < 0 || n_slots < 0 || (q && H < 1)) return fail(KDA_ERR_INVALID_ARGUMENT, "sizes out of range");
  if (N == 0) return KDA_OK;
  if (N > kMaxBlocks) return fail(KDA_ERR_UNSUPPORTED, "N=%d over %lld", N, static_cast<long long>(kMaxBlocks));
  if (!rows || !positions || !slots || !cos_sin || n_positions < 1) return fail(KDA_ERR_INVALID_ARGUMENT, "null rows, positions, slots or cos_sin");
  if (n_slots > 0 && !cache) return fail(KDA_ERR_INVALID_ARGUMENT, "null cache");
  if ((q == nullptr) != (q_out == nullptr)) return fail(KDA_ERR_INVALID_ARGUMENT, "q and q_out go together");
  if (norm_weight && !(eps >= 0.f)) return fail(KDA_ERR_INVALID_ARGUMENT, "eps must not be negative");
  const int64_t es = static_cast<int64_t>(elem(dtype));
  for (const void* p : {rows, static_cast<const void*>(cache), static_cast<const void*>(cos_sin), static_cast<const void*>(norm_weight)})
    if (!aligned(p, 16)) return fail(KDA_ERR_INVALID_ARGUMENT, "rows, cache, cos_sin and norm_weight must be aligned to 16 bytes");
  if (rows_stride < 0 || rows_stride * es % 16 != 0) return fail(KDA_ERR_INVALID_ARGUMENT, "rows_stride must be a multiple of 16 bytes");
  if (!aligned(q, 4 * es) || !aligned(q_out, 4 * es) || q_stride_t % 4 || q_stride_h % 4 || qo_stride_t % 4 || qo_stride_h % 4)
    return fail(KDA_ERR_INVALID_ARGUMENT, "q and q_out must be aligned to 4 elements, their strides too");
  kda::LatentAppendArgs a{};
  a.rows = rows; a.positions = positions; a.slots = slots; a.cos_sin = cos_sin; a.w = norm_weight;
  a.cache = cache; a.q = q; a.q_out = q_out;
  a.rows_t = rows_stride; a.q_t = q_stride_t; a.q_h = q_stride_h; a.qo_t = qo_stride_t; a.qo_h = qo_stride_h;
  a.n_slots = n_slots; a.P = n_positions; a.N = N; a.H = H; a.interleaved = interleaved != 0; a.eps = eps;
  return launched(kda::launch_latent_append(a, R, dr, dtype, stream), "kda_latent_append");
}

size_t kda_latent_decode_workspace(int B, int Tq, int H, int R, int dr, int page_size, int max_pages, int dtype) {
  DecodePlan P;
  if (B < 0 || Tq < 1 || H < 1 || (R != 256 && R != 512) || (dr != 32 && dr != 64) || !pow2(page_size) || max_pages < 0 ||
      !dtype_ok(dtype) || !decode_plan(B, Tq, H, R, page_size, max_pages, dtype, &P))
    return 0;
  return P.total;
}

int kda_latent_decode(hipStream_t stream, const void* q, const void* cache, const int32_t* block_table, const int32_t* seq_lens,
                      void* o, float* lse, int B, int Tq, int H, int R, int dr, int64_t n_pages, int page_size, int max_pages,
                      float scale, int dtype, void* workspace, size_t workspace_bytes) {
  if (!dtype_ok(dtype)) return fail(KDA_ERR_INVALID_ARGUMENT, "dtype=%d must be F32, BF16 or F16", dtype);
  if ((R != 256 && R != 512) || (dr != 32 && dr != 64))
    return fail(KDA_ERR_UNSUPPORTED, "R=%d, dr=%d unsupported (R in {256, 512}, dr in {32, 64})", R, dr);
  if (B < 0 || Tq < 1 || H < 1 || max_pages < 0 || n_pages < 0) return fail(KDA_ERR_INVALID_ARGUMENT, "sizes out of range");
  if (!pow2(page_size)) return fail(KDA_ERR_INVALID_ARGUMENT, "page_size=%d must be a power of two", page_size);
  if (n_pages >= (int64_t{1} << 31) / page_size) return fail(KDA_ERR_UNSUPPORTED, "n_pages * page_size must be below 2^31");
  if (B > 65535) return fail(KDA_ERR_UNSUPPORTED, "B=%d over 65535", B);
  if (!(scale > 0.f) || !std::isfinite(scale)) return fail(KDA_ERR_INVALID_ARGUMENT, "scale must be positive and finite");
  if (B == 0) return KDA_OK;
  if (n_pages == 0) max_pages = 0;      // no page: every length is 0
  if (!q || !seq_lens || !o || !lse || (max_pages > 0 && (!cache || !block_table)))
    return fail(KDA_ERR_INVALID_ARGUMENT, "null q, cache, block_table, seq_lens, o or lse");
  for (const void* p : {q, cache, static_cast<const void*>(o), static_cast<const void*>(workspace)})
    if (!aligned(p, 16)) return fail(KDA_ERR_INVALID_ARGUMENT, "q, cache, o and workspace must be aligned to 16 bytes");
  DecodePlan P;
  if (!decode_plan(B, Tq, H, R, page_size, max_pages, dtype, &P))
    return fail(KDA_ERR_UNSUPPORTED, "Tq * H = %lld rows or B * max_pages * page_size too large", static_cast<long long>(Tq) * H);
  if (!workspace || workspace_bytes < P.total)
    return fail(KDA_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : size_t{0}, P.total);
  kda::LatentDecodeArgs a{};
  a.q = q; a.cache = cache; a.table = block_table; a.lens = seq_lens; a.o = o; a.lse = lse;
  a.line = static_cast<int*>(workspace);
  a.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + P.part_ml);
  a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + P.part_o);
  a.B = B; a.Tq = Tq; a.H = H; a.per = max_pages; a.n_pages = n_pages;
  for (a.page_shift = 0; (1 << a.page_shift) < page_size;) ++a.page_shift;
  a.groups = P.groups; a.wgs = P.wgs; a.whole = P.whole; a.least = P.least; a.pad = P.pad; a.scale = scale;
  return launched(kda::launch_latent_decode(a, R, dr, dtype, P.rows, stream), "kda_latent_decode");
}

}  // extern "C"
