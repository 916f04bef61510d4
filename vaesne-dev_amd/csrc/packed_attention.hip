// Packed-sequence attention: argument checks, the choice of tiles and splits, the small kernels
// (packed_attention.h has the attention kernels, packed_attention_<type>.hip their instances).
#include <algorithm>

#include "packed_attention.h"

using namespace vaesne;
using namespace vaesne::pk;

namespace vaesne {
namespace pk {

template <> int run_fwd<float>(const Plan& p, hipStream_t s);
template <> int run_fwd<__bf16>(const Plan& p, hipStream_t s);
template <> int run_fwd<_Float16>(const Plan& p, hipStream_t s);
template <> int run_bwd<float>(const Plan& p, hipStream_t s);
template <> int run_bwd<__bf16>(const Plan& p, hipStream_t s);
template <> int run_bwd<_Float16>(const Plan& p, hipStream_t s);

__global__ __launch_bounds__(256) void add_parts_kernel(const float* part, int parts, int64_t n, float* out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float x = 0.f;
  for (int k = 0; k < parts; ++k) x += part[k * n + i];
  out[i] = x;
}

__global__ __launch_bounds__(1024) void hist_sum_kernel(const float* hist, int n, int Hq, int NH, float* rel) {
  __shared__ float part[16][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), slice = threadIdx.x >> 6, head = blockIdx.y;
  float x = 0.f;
  if (c < NH)
    for (int i = slice; i < n; i += 16) x += hist[((int64_t)i * Hq + head) * NH + c];
  part[slice][threadIdx.x & 63] = x;
  __syncthreads();
  if (slice == 0 && c < NH) {
    x = 0.f;
    for (int i = 0; i < 16; ++i) x += part[i][threadIdx.x];
    rel[(int64_t)head * NH + c] = x;
  }
}

namespace {

constexpr int CUS = 256;
constexpr int MAX_SPLIT = 64;
constexpr int ROW_TILES = 12;          // of a part of row_kernel's walk: its parts cost 4 bytes a row (8 to 16 are alike, 38 us; one part 48)
constexpr int64_t MAX_PART = 256 << 20;
constexpr int64_t MAX_STRIDE = 1 << 21;  // elements: a tile of 128 rows spans less than 2^31 bytes
constexpr int64_t MAX_TOKENS = (1 << 30) - 64;  // 4 threads of a launch each, 64 a workgroup; an axis of a grid has fewer than 2^32
constexpr int64_t MAX_ROWS = 1 << 25; // rows of one sequence: 32-bit row arithmetic with room

// Parts to cut the streamed axis into, in units of a tile (about 1.2 us).  Each of `wgs` workgroups walks
// up to `longest` tiles, `mean` on average; `slots` of them run at once, longest first, beside `beside`
// units of other work.  Parts have the same length for all (a shorter walk has fewer of them), cost about
// six tiles more each, and are written and read back once (4.5 TB/s) by a joining launch.  The end of the launch is estimated as
//   max(all tiles and parts / slots + beside + half of the longest part, the longest part) + joining
// and the fewest parts taken that come within a twentieth of the best.  (fp16 training, 6 sequences of up
// to 2047, 12 heads: one part 48 us forward, two 58 + 17 us; one token over 32 caches of up to 16384
// keys: one part 0.35 ms, as chosen 0.13.)
int splits(int64_t wgs, int64_t longest, double mean, int64_t part_bytes, int slots, double beside) {
  const double over = 6;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(MAX_SPLIT, longest / 4),
                                                              MAX_PART / std::max<int64_t>(part_bytes, 1)));
  auto end = [&](int64_t n) {
    const double own = (double)((longest + n - 1) / n) + over;
    const double join = n > 1 ? 4 + (double)n * part_bytes / 2.7e6 : 0;
    const double parts = std::max(1.0, n * mean / std::max<double>(longest, 1));
    return std::max(wgs * (mean + parts * over) / slots + beside + 0.5 * own, own) + join;
  };
  double least = end(1);
  for (int64_t n = 2; n <= most; ++n) least = std::min(least, end(n));
  for (int64_t n = 1; n < most; ++n)
    if (end(n) <= 1.05 * least) return (int)n;
  return (int)most;
}

int64_t up16(int64_t n) { return (n + 15) & ~(int64_t)15; }

bool sizes_ok(const vaesne_packed_attn* a) {
  return a && a->type >= 0 && a->type <= 2 && a->Hq > 0 && a->Hkv > 0 && a->Hq % a->Hkv == 0 && a->D > 0 &&
         a->D <= 128 && a->D % 8 == 0 && a->nseq >= 0 && a->max_q >= 0 && a->max_k >= 0 && a->total_q >= 0 &&
         a->total_k >= 0 && a->total_q <= MAX_TOKENS && a->total_k <= MAX_TOKENS && a->scale > 0.f && a->Hq <= 4096 &&
         (a->table == nullptr || (a->max_distance >= 1 && a->max_distance <= 512 && a->num_buckets >= 1));
}

// query heads of a key head that share a tile: the largest divisor of the group that a 64-row tile
// holds; one with a bias, whose table differs from head to head
int heads_per_tile(const vaesne_packed_attn* a) {
  if (a->table) return 1;
  const int g = a->Hq / a->Hkv;
  for (int p = std::min(g, 32); p > 1; --p)
    if (g % p == 0) return p;
  return 1;
}

// the same in dK / dV: a power of two, and no more than the rows between a thread's chunks
int log_heads_per_row_tile(const vaesne_packed_attn* a, int dp, int waves) {
  if (a->table) return 0;
  const int g = a->Hq / a->Hkv, rows = waves * 64 / (dp * (a->type == 0 ? 4 : 2) / 16);
  int l = 0;
  while (l < 5 && g % (2 << l) == 0 && (2 << l) <= rows) ++l;
  return l;
}

int waves_for(int64_t rows) { return rows <= 64 ? 2 : 4; }

int make_plan(const vaesne_packed_attn* a, int backward, Plan* p) {
  if (!sizes_ok(a)) return (int)hipErrorInvalidValue;
  *p = Plan{};
  Args& r = p->a;
  r.p = *a;
  r.group = a->Hq / a->Hkv;
  r.pg = heads_per_tile(a);
  r.nsub = r.group / r.pg;
  r.pgm = r.pg == 1 ? 0u : (uint32_t)(((1ull << 32) + r.pg - 1) / r.pg);
  if ((int64_t)a->max_q * r.pg > MAX_ROWS || (int64_t)a->max_k * r.pg > MAX_ROWS) return (int)hipErrorInvalidValue;
  r.c = a->scale * LOG2E;
  p->dp = a->D <= 16 ? 16 : a->D <= 32 ? 32 : a->D <= 64 ? 64 : 128;
  const int64_t rows = (int64_t)a->max_q * r.pg;
  p->nwk = waves_for(std::max<int64_t>(rows, a->max_k));
  p->nwq = backward ? p->nwk : waves_for(rows);
  r.pk_log = log_heads_per_row_tile(a, p->dp, p->nwk);
  r.nsubk = r.group >> r.pk_log;
  const int bn = a->type == 0 || (p->dp == 128 && p->nwq == 2) ? 32 : 64;   // key_tile()
  const int64_t qrows = a->total_q * a->Hq, krows = a->total_k * a->Hkv;
  const double n = std::max(a->nseq, 1);
  // a launch's workgroups of at most 256 threads: below 2^32 threads
  if (a->n_q_tiles < 0 || a->n_k_tiles < 0 || (int64_t)a->n_q_tiles * a->Hq >= (1 << 24) || (int64_t)a->n_k_tiles * a->Hkv >= (1 << 24))
    return (int)hipErrorInvalidValue;
  r.wgs_q = a->n_q_tiles * a->Hkv * r.nsub;
  r.wgs_k = backward ? a->n_k_tiles * a->Hkv : 0;
  const int bp = (a->type == 0 || p->dp == 128 ? 32 : 64) >> r.pk_log;     // row_tile()
  const double mean_q = a->total_k / n / bn, mean_k = (double)r.nsubk * a->total_q / n / bp;
  const int slots = CUS * (p->nwq == 2 ? 4 : 2);                 // workgroups that run at once
  const int64_t long_q = (a->max_k + bn - 1) / bn, long_k = (int64_t)r.nsubk * ((a->max_q + bp - 1) / bp);
  r.split_q = splits(r.wgs_q, long_q, mean_q, qrows * (a->D + 1) * 4, slots, r.wgs_k * mean_k / slots);
  r.split_k = splits(r.wgs_k, long_k, mean_k, 2 * krows * a->D * 4, slots, r.wgs_q * mean_q / slots);
  if (backward && ((int64_t)r.wgs_q * r.split_q + (int64_t)r.wgs_k * r.split_k) * p->nwk * 64 >= 1ll << 32)
    return (int)hipErrorInvalidValue;
  r.per_q = (int)((long_q + r.split_q - 1) / r.split_q);
  r.split_r = (int)std::max<int64_t>(1, std::min<int64_t>({(long_q + ROW_TILES - 1) / ROW_TILES, MAX_SPLIT, MAX_PART / std::max<int64_t>(qrows * 4, 1)}));
  r.per_r = (int)((long_q + r.split_r - 1) / r.split_r);
  r.per_k = (int)((long_k + r.split_k - 1) / r.split_k);
  return 0;
}

// the workspace: parts of the forward or dQ, their statistics | of dK / dV | rowsum(dO O) and its parts | bias sums
int64_t carve(Plan* p, int backward) {
  Args& r = p->a;
  const vaesne_packed_attn& a = r.p;
  const int64_t qrows = a.total_q * a.Hq, krows = a.total_k * a.Hkv, NH = 2 * a.max_distance + 1;
  const bool bias = backward && a.table && a.dtable;
  p->hist_bytes = bias ? up16((int64_t)a.n_q_tiles * a.Hq * r.split_q * NH * 4) : 0;
  int64_t used = 0;
  auto take = [&](int64_t bytes) {
    float* at = reinterpret_cast<float*>(reinterpret_cast<uintptr_t>(a.workspace) + used);
    used += up16(bytes);
    return at;
  };
  r.part = take(r.split_q > 1 ? r.split_q * qrows * a.D * 4 : 0);
  r.part_lse = take(!backward && r.split_q > 1 ? r.split_q * qrows * 4 : 0);
  r.part_k = take(backward && r.split_k > 1 ? 2 * r.split_k * krows * a.D * 4 : 0);
  r.delta = take(backward ? qrows * 4 : 0);
  r.part_delta = take(bias && a.type == 1 && r.split_r > 1 ? r.split_r * qrows * 4 : 0);
  r.hist = take(p->hist_bytes);
  take(bias ? (int64_t)a.Hq * NH * 4 : 0);                       // behind hist: its sums
  return used;
}

bool aligned(const void* p, int64_t ts, int64_t hs, int size) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ts * size) % 16 == 0 && (hs * size) % 16 == 0 && ts >= 0 && hs >= 0 &&
         ts < MAX_STRIDE && hs < MAX_STRIDE;
}

int check(const Plan& p, int64_t bytes, int backward) {
  const vaesne_packed_attn& a = p.a.p;
  const int size = a.type == 0 ? 4 : 2;
  const int bad = (int)hipErrorInvalidValue;
  if (a.q_tile != p.nwq * 32 / p.a.pg || (backward && a.k_tile != p.nwk * 32)) return bad;
  if ((a.total_q > 0 && (a.n_q_tiles == 0 || !a.q_tiles || !a.q || !a.o || !a.lse)) ||
      (a.total_k > 0 && (!a.k || !a.v)))
    return bad;
  if (!aligned(a.q, a.q_ts, a.q_hs, size) || !aligned(a.k, a.k_ts, a.k_hs, size) || !aligned(a.v, a.v_ts, a.v_hs, size) ||
      !aligned(a.o, 0, 0, size))
    return bad;
  if (a.table && !a.lut) return bad;
  if (bytes > 0 && (!a.workspace || (reinterpret_cast<uintptr_t>(a.workspace) & 15))) return bad;
  if (backward) {
    if (a.total_q > 0 && (!a.dout || !a.dq)) return bad;
    if (a.total_k > 0 && (!a.dk || !a.dv || a.n_k_tiles == 0 || !a.k_tiles)) return bad;
    if (!aligned(a.dout, a.do_ts, a.do_hs, size) || !aligned(a.dq, 0, 0, size) || !aligned(a.dk, 0, 0, size) ||
        !aligned(a.dv, 0, 0, size))
      return bad;
  }
  return 0;
}

}  // namespace
}  // namespace pk
}  // namespace vaesne

VAESNE_API int vaesne_packed_attn_tiles(const vaesne_packed_attn* a, int backward, int* q_tile, int* k_tile) {
  Plan p;
  const int rc = make_plan(a, backward, &p);
  if (rc) return rc;
  *q_tile = p.nwq * 32 / p.a.pg;
  *k_tile = p.nwk * 32;
  return 0;
}

VAESNE_API int64_t vaesne_packed_attn_workspace(const vaesne_packed_attn* a, int backward) {
  Plan p;
  if (make_plan(a, backward, &p)) return -1;
  return carve(&p, backward);
}

VAESNE_API int vaesne_packed_attn_fwd(const vaesne_packed_attn* a, void* stream) {
  Plan p;
  int rc = make_plan(a, 0, &p);
  if (!rc) rc = check(p, carve(&p, 0), 0);
  if (rc || a->total_q == 0) return rc;
  hipStream_t s = (hipStream_t)stream;
  return a->type == 0 ? run_fwd<float>(p, s) : a->type == 1 ? run_fwd<__bf16>(p, s) : run_fwd<_Float16>(p, s);
}

VAESNE_API int vaesne_packed_attn_bwd(const vaesne_packed_attn* a, void* stream) {
  Plan p;
  int rc = make_plan(a, 1, &p);
  if (!rc) rc = check(p, carve(&p, 1), 1);
  if (rc) return rc;
  hipStream_t s = (hipStream_t)stream;
  return a->type == 0 ? run_bwd<float>(p, s) : a->type == 1 ? run_bwd<__bf16>(p, s) : run_bwd<_Float16>(p, s);
}
