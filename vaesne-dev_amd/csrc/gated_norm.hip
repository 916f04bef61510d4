// The join between two blocks (include/vaesne_hip.h: vaesne_gated_norm): the norm after a block, its
// gate, the scaled residual and the norm before the next block in one pass over the rows.
//   u = N(f) w1 + b1,  y = c x + g u,  n = N(y) w2 + b2
// P threads hold a row in registers (NV chunks of V elements each), so every statistic is taken in
// two steps (mean, then squares of the differences) from one read.  Backward, with fh = N(f), yh = N(y):
//   G = dy + N'(dn w2),  dx = c G,  e = G g,  df = N'(e w1)
//   N'(d) = rstd (d - hat mean(d hat) [- mean(d)])
//   dw2 = sum dn yh, db2 = sum dn, dg = G u (summed over the rows for a channel gate), dw1 = sum e fh,
//   db1 = sum e
// y is computed again from x and f (the same bytes as reading it back, and unrounded).  A workgroup
// walks rows and keeps its columns' parameter sums in fp32 registers; the workgroups' partial sums
// are added in a fixed order.  Bound by HBM: forward 4, backward 6 passes over [rows, C], 5 and 8 with a gate per
// token (16384 x 4096 bf16, such a gate: 118 and 240 us, 5.7 and 4.5 TB/s; a copy of 1 GiB reaches 5.2).
#include <algorithm>

#include "common.h"

using namespace vaesne;

namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// threads of a workgroup: a row's, at least 256 (smaller rows share one)
template <int P> constexpr int NT = P > 256 ? P : 256;
template <int P> constexpr bool WHOLE = P >= 256;      // one row per workgroup

// V elements of T as loaded
template <class T, int V> struct Raw {
  u4 r;
  __device__ __forceinline__ void load(const T* p) { r = *reinterpret_cast<const u4*>(p); }
};
template <class T> struct Raw<T, 1> {
  T r;
  __device__ __forceinline__ void load(const T* p) { r = *p; }
};

// V elements of T as fp32; V = 1 for widths or alignments that do not allow 16-byte chunks
template <class T, int V> struct Chunk {
  float v[V];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V == 1) {
      v[0] = (float)p[0];
    } else {
      const u4 r = *reinterpret_cast<const u4*>(p);
      T t[V];
      __builtin_memcpy(t, &r, 16);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = (float)t[e];
    }
  }
  __device__ __forceinline__ void take(const Raw<T, V>& x) {
    T t[V];
    __builtin_memcpy(t, &x.r, sizeof(t));
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (float)t[e];
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V == 1) {
      p[0] = (T)v[0];
    } else {
      T t[V];
#pragma unroll
      for (int e = 0; e < V; ++e) t[e] = (T)v[e];
      u4 r;
      __builtin_memcpy(&r, t, 16);
      *reinterpret_cast<u4*>(p) = r;
    }
  }
  __device__ __forceinline__ void fill(float x) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = x;
  }
};

// sum over a workgroup's waves' values in LDS, in order
template <int P> __device__ __forceinline__ float lds_sum(const float* buf) {
  float x = buf[0];
#pragma unroll
  for (int i = 1; i < P / 64; ++i) x += buf[i];
  return x;
}

// sum over the P threads of a row; a whole workgroup's goes through LDS (`buf`: 8 floats, not the last call's)
template <int P> __device__ __forceinline__ float row_sum(float x, float* buf) {
  if constexpr (P == 8) {
    x += dpp_mov<0xb1>(x);
    x += dpp_mov<0x4e>(x);
    x += dpp_mov<0x141>(x);                           // half-row mirror: the other quad of the 8 lanes
    return x;
  } else {
    x = wave_sum(x);
    if constexpr (WHOLE<P>) {
      if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = x;
      __syncthreads();
      x = lds_sum<P>(buf);
    }
    return x;
  }
}

struct NArgs {
  vaesne_gated_norm p;
  float* partial;      // [workgroups][5][C]: pre_w, post_w, gate, pre_b, post_b
};

template <class T> __device__ __forceinline__ const T* row_at(const void* p, int64_t r, int64_t ld) {
  return reinterpret_cast<const T*>(p) + r * ld;
}

// mean and 1 / std of the row held in v (absent columns hold 0)
template <class T, int P, int V, int NV>
__device__ __forceinline__ void stats_of(const Chunk<T, V> (&v)[NV], int C, int tid, bool layer, float eps, float* red,
                                         float& mean, float& rstd) {
  mean = 0.f;
  if (layer) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) s += v[i].v[e];
    mean = row_sum<P>(s, red) / (float)C;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((i * P + tid) * V < C)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = v[i].v[e] - mean;
        q = fmaf(d, d, q);
      }
  // 1 / sqrt: the root and the quotient are rounded once each
  rstd = 1.f / sqrtf(row_sum<P>(q, red + 8) / (float)C + eps);
}

template <class T, int P, int V, int NV> __global__ __launch_bounds__(NT<P>) void fwd_kernel(NArgs a) {
  __shared__ float red[32];
  constexpr int RPB = NT<P> / P;
  const vaesne_gated_norm& p = a.p;
  const int tid = threadIdx.x % P, C = p.C;
  const int64_t r = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * RPB + threadIdx.x / P;
  const bool live = r < p.rows, layer = p.kind == 1;
  if (WHOLE<P> && !live) return;                       // (whole workgroups only)
  Chunk<T, V> x[NV], f[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * P + tid) * V;
    x[i].fill(0.f);
    f[i].fill(0.f);
    if (live && c < C) {
      x[i].load(row_at<T>(p.x, r, p.ldx) + c);
      if (p.branch) f[i].load(row_at<T>(p.branch, r, p.ldbranch) + c);
    }
  }
  float m1 = 0.f, r1 = 0.f, m2, r2;
  if (p.branch) stats_of<T, P, V, NV>(f, C, tid, layer, p.eps, red, m1, r1);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * P + tid) * V;
    if (!live || c >= C) continue;
#pragma unroll
    for (int e = 0; e < V; ++e) x[i].v[e] *= p.residual_scale;
    if (p.branch) {
      Chunk<T, V> w, b, g;
      w.load(row_at<T>(p.post_w, 0, 0) + c);
      b.fill(0.f);
      g.fill(1.f);
      if (p.post_b) b.load(row_at<T>(p.post_b, 0, 0) + c);
      if (p.gate_kind) g.load(row_at<T>(p.gate, p.gate_kind == 2 ? r : 0, p.ldgate) + c);
#pragma unroll
      for (int e = 0; e < V; ++e) x[i].v[e] = fmaf(g.v[e], fmaf((f[i].v[e] - m1) * r1, w.v[e], b.v[e]), x[i].v[e]);
    }
    if (p.y) x[i].store(reinterpret_cast<T*>(p.y) + r * C + c);
  }
  stats_of<T, P, V, NV>(x, C, tid, layer, p.eps, red + 16, m2, r2);
  if (!live) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * P + tid) * V;
    if (c >= C) continue;
    Chunk<T, V> w, b;
    w.load(row_at<T>(p.pre_w, 0, 0) + c);
    b.fill(0.f);
    if (p.pre_b) b.load(row_at<T>(p.pre_b, 0, 0) + c);
#pragma unroll
    for (int e = 0; e < V; ++e) w.v[e] = fmaf((x[i].v[e] - m2) * r2, w.v[e], b.v[e]);
    w.store(reinterpret_cast<T*>(p.n) + r * C + c);
  }
  if (p.stats && tid == 0) *reinterpret_cast<float4*>(p.stats + 4 * r) = make_float4(m1, r1, m2, r2);
}

// d -> rstd (d - hat mean(d hat) [- mean(d)]), both row sums at once
template <class T, int P, int V, int NV, bool LAYER>
__device__ __forceinline__ void norm_back(Chunk<T, V> (&d)[NV], const Chunk<T, V> (&hat)[NV], float rstd, int C, float* red) {
  float s = 0.f, q = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (LAYER) s += d[i].v[e];
      q = fmaf(d[i].v[e], hat[i].v[e], q);
    }
  if constexpr (WHOLE<P>) {
    if (LAYER) s = wave_sum(s);
    q = wave_sum(q);
    if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = q; if (LAYER) red[8 + (threadIdx.x >> 6)] = s; }
    __syncthreads();
    q = lds_sum<P>(red);
    if (LAYER) s = lds_sum<P>(red + 8);
  } else {
    if (LAYER) s = row_sum<P>(s, red);
    q = row_sum<P>(q, red);
  }
  s /= (float)C;
  q /= (float)C;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) d[i].v[e] = rstd * (d[i].v[e] - hat[i].v[e] * q - (LAYER ? s : 0.f));
}

template <class T, int P, int V, int NV, bool LAYER> __global__ __launch_bounds__(NT<P>) void bwd_kernel(NArgs a) {
  constexpr int RPB = NT<P> / P, K = LAYER ? 5 : 3, COLS = P * V * NV;
  __shared__ float red[32];
  __shared__ float sums[WHOLE<P> ? 1 : 4 * COLS];
  const vaesne_gated_norm& p = a.p;
  const int tid = threadIdx.x % P, C = p.C;
  const float cs = p.residual_scale;
  float acc[K][NV][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) acc[k][i][e] = 0.f;
  // the next turn's rows are in flight during this turn's sums (without: 309 us at 16384 x 4096 bf16
  // with a gate per token, with: 238 us)
  Raw<T, V> rx[NV], rf[NV], rd[NV], rG[NV], rg[NV];
  float4 rst = make_float4(0.f, 0.f, 0.f, 0.f);
  auto fetch = [&](int64_t r) {
    if (r >= p.rows) return;
    rst = *reinterpret_cast<const float4*>(p.stats + 4 * r);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * P + tid) * V;
      if (c >= C) continue;
      rx[i].load(row_at<T>(p.x, r, p.ldx) + c);
      if (p.branch) rf[i].load(row_at<T>(p.branch, r, p.ldbranch) + c);
      if (p.gate_kind == 2) rg[i].load(row_at<T>(p.gate, r, p.ldgate) + c);
      if (p.dy) rG[i].load(row_at<T>(p.dy, r, p.lddy) + c);
      if (p.dn) rd[i].load(row_at<T>(p.dn, r, p.lddn) + c);
    }
  };
  constexpr bool AHEAD = V > 1 && NV < 4;             // (single elements and 4 chunks: it spills)
  const int64_t turn = (int64_t)gridDim.x * RPB;
  if (AHEAD) fetch((int64_t)blockIdx.x * RPB + threadIdx.x / P);
  // every thread of a workgroup takes the same number of turns (the row sums hold barriers)
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < p.rows; r0 += turn) {
    const int64_t r = r0 + threadIdx.x / P;
    const bool live = r < p.rows;
    float4 st = rst;
    if (!AHEAD && live) st = *reinterpret_cast<const float4*>(p.stats + 4 * r);
    Chunk<T, V> fh[NV], yh[NV], d[NV], g[NV], G[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * P + tid) * V;
      fh[i].fill(0.f); yh[i].fill(0.f); d[i].fill(0.f); g[i].fill(0.f); G[i].fill(0.f);
      if (!live || c >= C) continue;
      if (AHEAD) {
        yh[i].take(rx[i]);
        if (p.branch) fh[i].take(rf[i]);
        if (p.gate_kind == 2) g[i].take(rg[i]);
        if (p.dy) G[i].take(rG[i]);
        if (p.dn) d[i].take(rd[i]);
      } else {
        yh[i].load(row_at<T>(p.x, r, p.ldx) + c);
        if (p.branch) fh[i].load(row_at<T>(p.branch, r, p.ldbranch) + c);
        if (p.gate_kind == 2) g[i].load(row_at<T>(p.gate, r, p.ldgate) + c);
        if (p.dy) G[i].load(row_at<T>(p.dy, r, p.lddy) + c);
        if (p.dn) d[i].load(row_at<T>(p.dn, r, p.lddn) + c);
      }
    }
    if (AHEAD) fetch(r + turn);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * P + tid) * V;
      if (!live || c >= C) continue;
      Chunk<T, V> w, b;
#pragma unroll
      for (int e = 0; e < V; ++e) yh[i].v[e] *= cs;
      if (p.branch) {
        w.load(row_at<T>(p.post_w, 0, 0) + c);
        b.fill(0.f);
        if (LAYER && p.post_b) b.load(row_at<T>(p.post_b, 0, 0) + c);
        if (p.gate_kind == 0) g[i].fill(1.f);
        if (p.gate_kind == 1) g[i].load(row_at<T>(p.gate, 0, 0) + c);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          fh[i].v[e] = (fh[i].v[e] - st.x) * st.y;
          yh[i].v[e] = fmaf(g[i].v[e], fmaf(fh[i].v[e], w.v[e], b.v[e]), yh[i].v[e]);
        }
      }
      w.load(row_at<T>(p.pre_w, 0, 0) + c);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        yh[i].v[e] = (yh[i].v[e] - st.z) * st.w;
        acc[0][i][e] = fmaf(d[i].v[e], yh[i].v[e], acc[0][i][e]);
        if (LAYER) acc[3][i][e] += d[i].v[e];
        d[i].v[e] *= w.v[e];
      }
    }
    norm_back<T, P, V, NV, LAYER>(d, yh, st.w, C, red);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * P + tid) * V;
      if (!live || c >= C) { d[i].fill(0.f); continue; }
      Chunk<T, V> w, b, o;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        G[i].v[e] += d[i].v[e];
        o.v[e] = G[i].v[e] * cs;
      }
      o.store(reinterpret_cast<T*>(p.dx) + r * C + c);
      if (!p.branch) { d[i].fill(0.f); continue; }
      w.load(row_at<T>(p.post_w, 0, 0) + c);
      b.fill(0.f);
      if (LAYER && p.post_b) b.load(row_at<T>(p.post_b, 0, 0) + c);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float e1 = G[i].v[e] * g[i].v[e];
        o.v[e] = G[i].v[e] * fmaf(fh[i].v[e], w.v[e], b.v[e]);       // dgate
        acc[2][i][e] += o.v[e];
        acc[1][i][e] = fmaf(e1, fh[i].v[e], acc[1][i][e]);
        if (LAYER) acc[4][i][e] += e1;
        d[i].v[e] = e1 * w.v[e];
      }
      if (p.gate_kind == 2 && p.dgate) o.store(reinterpret_cast<T*>(p.dgate) + r * C + c);
    }
    if (p.branch) {
      norm_back<T, P, V, NV, LAYER>(d, fh, st.y, C, red + 16);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * P + tid) * V;
        if (live && c < C) d[i].store(reinterpret_cast<T*>(p.dbranch) + r * C + c);
      }
    } else if (WHOLE<P>) {
      __syncthreads();                                // the next row's sums reuse red[0..15]
    }
  }
  // this workgroup's column sums, rows of the same column added in a fixed order
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float* out = a.partial + ((int64_t)blockIdx.x * 5 + k) * C;
    if constexpr (WHOLE<P>) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int c = (i * P + tid) * V + e;
          if (c < C) out[c] = acc[k][i][e];
        }
    } else {
      __syncthreads();
      float* mine = sums + (threadIdx.x >> 6) * COLS;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float x = acc[k][i][e];
          if constexpr (P == 8) {                     // the 8 row groups of a wave
            x += dpp_mov<0x128>(x);
            x = xsum32(xsum16(x));
          }
          if ((threadIdx.x & 63) < P) mine[(i * P + tid) * V + e] = x;
        }
      __syncthreads();
      for (int c = threadIdx.x; c < C; c += NT<P>) out[c] = (sums[c] + sums[COLS + c]) + (sums[2 * COLS + c] + sums[3 * COLS + c]);
    }
  }
}

struct Outs { void* o[5]; };
// parameter gradients from the workgroups' partial sums: 32 columns, 32 slices of the workgroups in
// order, then the slices in order (25 MB of partial sums at 4096 columns: 7.5 us; 64 columns and 16
// slices leave CUs without a workgroup: 11.5)
template <class T> __global__ __launch_bounds__(1024) void param_kernel(const float* partial, int G, int C, Outs outs) {
  T* out = reinterpret_cast<T*>(outs.o[blockIdx.y]);
  if (!out) return;
  __shared__ float part[32][32];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
  float x = 0.f;
  if (c < C)
    for (int g = slice; g < G; g += 32) x += partial[((int64_t)g * 5 + blockIdx.y) * C + c];
  part[slice][threadIdx.x & 31] = x;
  __syncthreads();
  if (slice == 0 && c < C) {
    x = 0.f;
    for (int i = 0; i < 32; ++i) x += part[i][threadIdx.x];
    out[c] = (T)x;
  }
}

// threads per row: 8 for the models' own widths, a wave, then a workgroup; at most 16 columns each (with 32
// the backward's sums and the rows ahead spill).  A row of 256 to 512 chunks: one chunk a thread in the
// forward (16384 x 4096 bf16: 118 us, two 123), two in the backward (240 us, one 256: eight waves wait on every sum)
struct Shape { int V, P, NV; };
Shape shape_of(int C, int V, bool backward) {
  const int n = (C + V - 1) / V;
  if (V > 1 && n <= 8) return {V, 8, 1};
  if (V == 1) return n <= 256 ? Shape{1, 64, 4} : n <= 2048 ? Shape{1, 256, 8} : Shape{1, 512, 16};
  if (n <= 64) return {V, 64, 1};
  if (n <= 128) return {V, 64, 2};
  if (n <= 256) return {V, V == 4 ? 64 : 256, V == 4 ? 4 : 1};
  if (n <= 512) return backward ? Shape{V, 256, 2} : Shape{V, 512, 1};
  return n <= 1024 ? Shape{V, 512, 2} : Shape{V, 512, 4};
}
int groups_of(const vaesne_gated_norm& a, int P) {
  const int64_t rpb = P > 256 ? 1 : 256 / P;
  return (int)std::max<int64_t>(1, std::min<int64_t>(512, (a.rows + rpb - 1) / rpb));
}

bool bad(const vaesne_gated_norm* a) {
  return !a || (reinterpret_cast<uintptr_t>(a->stats) & 15) || a->type < 0 || a->type > 2 || a->kind < 0 || a->kind > 1 || a->gate_kind < 0 || a->gate_kind > 2 ||
         a->C < 1 || a->C > 8192 || a->rows < 0 || a->rows >= (1ll << 31);
}

// 16-byte chunks need every row of every tensor on a 16-byte boundary
int chunk_of(const vaesne_gated_norm& a) {
  const int size = a.type == 0 ? 4 : 2, V = 16 / size;
  uintptr_t m = 0;
  for (const void* q : {a.x, a.branch, a.gate, a.pre_w, a.pre_b, a.post_w, a.post_b, (const void*)a.y, (const void*)a.n,
                        a.dy, a.dn, (const void*)a.dx, (const void*)a.dbranch, (const void*)a.dgate})
    m |= reinterpret_cast<uintptr_t>(q);
  const int64_t l = a.ldx | a.ldbranch | a.ldgate | a.lddy | a.lddn | a.C;
  return (m & 15) == 0 && l % V == 0 ? V : 1;
}

template <class T, int P, int V, int NV> int go_fwd(const NArgs& a, hipStream_t s) {
  const int64_t rpb = NT<P> / P;
  // (an axis of a grid has fewer than 2^32 threads: workgroups past 2^22 go to the second)
  const int64_t wgs = (a.p.rows + rpb - 1) / rpb, wide = std::min<int64_t>(wgs, 1 << 22);
  hipLaunchKernelGGL((fwd_kernel<T, P, V, NV>), dim3((unsigned)wide, (unsigned)((wgs + wide - 1) / wide)), dim3(NT<P>), 0, s, a);
  VAESNE_CHECK_LAUNCH();
  return 0;
}

template <class T, int P, int V, int NV> int go_bwd(const NArgs& a, hipStream_t s) {
  const int G = groups_of(a.p, P);
  if (a.p.kind) hipLaunchKernelGGL((bwd_kernel<T, P, V, NV, true>), dim3(G), dim3(NT<P>), 0, s, a);
  else hipLaunchKernelGGL((bwd_kernel<T, P, V, NV, false>), dim3(G), dim3(NT<P>), 0, s, a);
  VAESNE_CHECK_LAUNCH();
  Outs o = {{a.p.dpre_w, a.p.dpost_w, a.p.gate_kind == 1 ? a.p.dgate : nullptr, a.p.kind ? a.p.dpre_b : nullptr,
             a.p.kind ? a.p.dpost_b : nullptr}};
  hipLaunchKernelGGL((param_kernel<T>), dim3((a.p.C + 31) / 32, a.p.kind ? 5 : 3), dim3(1024), 0, s, a.partial, G, a.p.C, o);
  VAESNE_CHECK_LAUNCH();
  return 0;
}

template <class T> int run(const vaesne_gated_norm& p, bool backward, hipStream_t s) {
  constexpr int W = 16 / sizeof(T);
  const NArgs a{p, reinterpret_cast<float*>(p.workspace)};
  const Shape q = shape_of(p.C, chunk_of(p), backward);
#define VAESNE_GN_FWD(PV, VV, NVV) if (!backward && q.P == PV && q.V == VV && q.NV == NVV) return go_fwd<T, PV, VV, NVV>(a, s);
#define VAESNE_GN_BWD(PV, VV, NVV) if (backward && q.P == PV && q.V == VV && q.NV == NVV) return go_bwd<T, PV, VV, NVV>(a, s);
#define VAESNE_GN(PV, VV, NVV) VAESNE_GN_FWD(PV, VV, NVV) VAESNE_GN_BWD(PV, VV, NVV)
  VAESNE_GN(8, W, 1) VAESNE_GN(64, W, 1) VAESNE_GN(64, W, 2) VAESNE_GN_FWD(512, W, 1) VAESNE_GN_BWD(256, W, 2) VAESNE_GN(512, W, 2)
  if constexpr (W == 4) { VAESNE_GN(64, W, 4) VAESNE_GN(512, W, 4) }
  else { VAESNE_GN(256, W, 1) }
  VAESNE_GN(64, 1, 4) VAESNE_GN(256, 1, 8) VAESNE_GN(512, 1, 16)
#undef VAESNE_GN
#undef VAESNE_GN_BWD
#undef VAESNE_GN_FWD
  return (int)hipErrorInvalidValue;
}

int dispatch(const vaesne_gated_norm* a, bool backward, void* stream) {
  hipStream_t s = (hipStream_t)stream;
  return a->type == 0 ? run<float>(*a, backward, s) : a->type == 1 ? run<__bf16>(*a, backward, s) : run<_Float16>(*a, backward, s);
}

}  // namespace

VAESNE_API int64_t vaesne_gated_norm_workspace(const vaesne_gated_norm* a) {
  if (bad(a)) return -1;
  // the most workgroups any chunk width gives: 8 threads per row never give more than a whole one
  return (int64_t)groups_of(*a, 256) * 5 * a->C * 4;
}

VAESNE_API int vaesne_gated_norm_fwd(const vaesne_gated_norm* a, void* stream) {
  if (bad(a)) return (int)hipErrorInvalidValue;
  if (a->rows == 0) return 0;
  if (!a->x || !a->n || !a->pre_w || (a->branch && (!a->y || !a->post_w)) || (a->gate_kind && (!a->gate || !a->branch)))
    return (int)hipErrorInvalidValue;
  return dispatch(a, false, stream);
}

VAESNE_API int vaesne_gated_norm_bwd(const vaesne_gated_norm* a, void* stream) {
  if (bad(a)) return (int)hipErrorInvalidValue;
  if (!a->workspace || (a->rows > 0 && (!a->x || !a->dx || !a->stats || !a->pre_w || (a->branch && (!a->dbranch || !a->post_w)) ||
                                        (a->gate_kind && (!a->gate || !a->branch)))))
    return (int)hipErrorInvalidValue;
  return dispatch(a, true, stream);
}
