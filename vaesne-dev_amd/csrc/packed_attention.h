// Attention over packed sequences (include/vaesne_hip.h: vaesne_packed_attn): one pass over the
// keys with a running maximum and sum, every product on the matrix cores, for fp32, bf16 and fp16.
//
// Layout of the products.  All tiles are 32x32 accumulators (v_mfma_f32_32x32x16_{bf16,f16}, and
// v_mfma_f32_32x32x2_f32 for fp32), and every one is oriented so that a lane owns one COLUMN: a
// query in the forward and in dQ, a key in dK / dV.  The forward computes S^T = K Q^T (rows are
// keys): a lane holds 16 scores of its own query, so the softmax needs one cross-lane exchange (lane
// l and l ^ 32 share a query) per key tile.  The contraction of the next product runs over those
// same rows (O^T = V^T P^T): a contraction may number its slots as it likes so long as both operands
// agree, so the accumulator registers of P are, in order, the other operand's slots
//     slot (half h, element j) of block t  <->  row  KC t + 8 (j / 4) + 4 h + j % 4
// and V^T is read from the row-major LDS tile with that numbering (ds_read_b64_tr_b16 for 16-bit
// types: 4 rows of one column per lane; four ds_read_b32 for fp32).  P never passes through LDS.
// The backward repeats the scheme: dQ^T = K^T dS^T beside S^T and dP^T = V dO^T, and, with a key per
// lane, dV^T = dO^T P and dK^T = Q^T dS beside S = Q K^T and dP = dO V^T.  dQ and dK / dV are two
// bodies of one launch that each compute S and dP (seven products instead of five): no atomic sums, so
// every gradient is bitwise reproducible.
//
// Measured (a product of 8192^3 reaches 1.2 PFLOP/s in bf16, 1.16 in fp16; a copy of 1 GiB 5.2 TB/s): three prompts
// of 2000 to 8001 tokens, causal, 32 heads of 128 over 8, bf16, 0.74 TFLOP without the masked half: 0.75 ms, 0.98 PFLOP/s;
// one new token over 32 caches, 0.43 GB of keys and values: 0.10 ms, 4.3 TB/s.  A kernel of many scores with a bias
// at head_dim 64 spends most on the vector ALUs (exp2, the maximum, the bias read per score; 70 % busy).
//
// LDS tiles are rows of DP elements in 16-byte chunks, chunk c of row r at c ^ swz(r): both the row
// reads (16 lanes: 16 rows of one chunk) and the transposed reads (32 lanes: 4 rows of 4 chunks)
// then touch all 64 banks once.  Rows outside a sequence and columns past D are zero, so nothing
// that lies behind a sequence can reach it.
//
// Grouped heads.  The PG query heads that share a key head are rows of one tile (row = position *
// PG + head), so K and V are read once for all of them, and one new token fills PG rows, not one.
// With few tiles the keys (forward, dQ) or the query rows (dK / dV) are split over workgroups, the
// parts kept in fp32 in the workspace and joined in a fixed order.
#pragma once
#include "common.h"

namespace vaesne {
namespace pk {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

template <class T> struct Ty;
template <> struct Ty<float> { using Frag = f4; using Quad = f4; };
template <> struct Ty<__bf16> { using Frag = b8; using Quad = b4; };
template <> struct Ty<_Float16> { using Frag = h8; using Quad = h4; };

constexpr float LOG2E = 1.4426950408889634f;
constexpr float INF = __builtin_inff();

struct Args {
  vaesne_packed_attn p;
  int pg, nsub, group;         // heads per tile, tiles per key head's group, query heads per key head
  int pk_log, nsubk;           // dK / dV: log2(heads per row tile), tiles per group
  uint32_t pgm;                // ceil(2^32 / pg), 0 for pg = 1
  int split_q, split_k;        // parts of the keys (forward, dQ), of the query rows (dK / dV)
  int split_r, per_r;          // row_kernel: parts of the keys, tiles of one
  int per_q, per_k;            // tiles of a part: the same for every sequence, short ones have fewer parts
  int wgs_q, wgs_k;            // workgroups of a part
  float c;                     // scale * log2(e)
  float* part;                 // the forward's or dQ's parts: [split_q][rows][D]
  float* part_k;               // dk parts [split_k][rows][D], then dv parts
  float* part_lse;             // [split_q][rows]
  float* delta;                // [total_q][Hq]: rowsum(dO O), or rowsum(P dP) (row_kernel)
  float* part_delta;           // its parts: [split_r][total_q][Hq]
  float* hist;                 // [dQ workgroups][2R + 1]
};

__device__ __forceinline__ int div_pg(const Args& a, int row) {
  return a.pgm ? (int)__umulhi((uint32_t)row, a.pgm) : row;
}

// ---- products ------------------------------------------------------------------------------
__device__ __forceinline__ f16v mma(b8 a, b8 b, f16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f16v mma(h8 a, h8 b, f16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f16v mma(f4 a, f4 b, f16v c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// accumulator registers of contraction block t as the other operand's fragment.  16-bit types
// round to nearest even here: P <= 2^8 (fp16 2^15) and dS enter the matrix cores in the inputs' own type, the
// sums stay fp32 (a relative 2^-8 (bf16), 2^-11 (fp16) of each term at most, independent between terms)
template <class T> __device__ __forceinline__ typename Ty<T>::Frag take(const f16v& s, int t) {
  constexpr int N = 16 / sizeof(T);
  float __attribute__((ext_vector_type(N))) v;
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = s[N * t + j];
  return __builtin_convertvector(v, typename Ty<T>::Frag);
}

// what take() left behind, for a second product
template <class T> __device__ __forceinline__ typename Ty<T>::Frag rest_of(const f16v& s, int t, const typename Ty<T>::Frag& taken) {
  constexpr int N = 16 / sizeof(T);
  float __attribute__((ext_vector_type(N))) v;
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = s[N * t + j] - (float)taken[j];
  return __builtin_convertvector(v, typename Ty<T>::Frag);
}

// ---- LDS tiles -----------------------------------------------------------------------------
template <class T, int DP> struct Tile {
  using Type = T;
  static constexpr int EPC = 16 / sizeof(T);          // elements per chunk
  static constexpr int CPR = DP / EPC;                // chunks per row
  static constexpr int RB = CPR * 16;                 // bytes per row
  static constexpr int KC = 2 * EPC;                  // depth of one fragment product
  static constexpr int NCH = DP / KC;                 // fragments per row
  static constexpr int DT = (DP + 31) / 32;           // 32-column tiles
  static constexpr int TB = 32 / KC;                  // contraction blocks per 32 rows
  static constexpr int CR = sizeof(T) == 2 ? 2 : 4;   // LDS reads of a transposed fragment

  static __device__ __forceinline__ int swz(int r) {
    if constexpr (CPR >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (CPR == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else if constexpr (CPR == 4) return (r >> 2) & 3;
    else return (r >> 3) & 1;
  }
  static __device__ __forceinline__ int at(int r, int c) { return r * RB + ((c ^ swz(r)) << 4); }

  // A lane's LDS offsets.  swz is a combination of xors of row bits, so a fragment's address is one
  // of these, xor a constant, plus a constant (a multiple of 16 rows, the tile): nothing but the
  // offsets stays in registers.  (Addresses kept for every fragment took 24 registers of each wave.)
  struct Lane {
    uint32_t r, c[2];
    __device__ __forceinline__ Lane(int lane) {
      const int h = lane >> 5, i = lane & 15;
      r = at(lane & 31, h);
      if constexpr (sizeof(T) == 2) {
        const int ch = (2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) & (CPR - 1);
#pragma unroll
        for (int j = 0; j < 2; ++j) c[j] = at(8 * j + 4 * h + (i >> 2), ch) + 8 * (i & 1);
      } else {
        c[0] = at(4 * h, ((lane & 31) >> 2) & (CPR - 1)) + 4 * (lane & 3);
        c[1] = 0;
      }
    }
    // not known to be the same from one tile to the next: the xors are taken again, not kept
    __device__ __forceinline__ void renew() { asm volatile("" : "+v"(r), "+v"(c[0]), "+v"(c[1])); }
  };
  // fragment of row r0 + lane % 32 (r0: a multiple of 32): columns KC k + EPC h ..
  static __device__ __forceinline__ typename Ty<T>::Frag row(const char* s, const Lane& l, int r0, int k) {
    return *reinterpret_cast<const typename Ty<T>::Frag*>(s + r0 * RB + (l.r ^ (k << 5)));
  }
  // transposed fragment: column 32 dt + lane % 32 of rows r0 + (block t's slots)
  static __device__ __forceinline__ typename Ty<T>::Frag col(const char* s, const Lane& l, int r0, int t, int dt) {
    if constexpr (sizeof(T) == 2) {
      u4 o;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s4*)(s + (r0 + KC * t) * RB + (l.c[j] ^ (CPR > 4 ? dt << 6 : 0))));
        const uint2 y = __builtin_bit_cast(uint2, x);
        o[2 * j] = y.x; o[2 * j + 1] = y.y;
      }
      return __builtin_bit_cast(typename Ty<T>::Frag, o);
    } else {
      typename Ty<T>::Frag o;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int f = (CPR >= 16 ? j << 2 : CPR == 8 ? (j >> 1) << 2 : 0) ^ (2 * (t & 1)) ^ (CPR > 8 ? 8 * dt : 0);
        o[j] = *reinterpret_cast<const float*>(s + (r0 + KC * t + j) * RB + (l.c[0] ^ (f << 4)));
      }
      return o;
    }
  }
};

// ROWS rows of a tile, global -> registers -> LDS (16-byte chunks; absent ones are zero).  A thread's
// offsets from the tile's first row never change, so a tile costs one buffer descriptor (scalar) and
// no address arithmetic; an absent chunk's offset lies outside the descriptor and reads as zero.
// (With 64-bit addresses computed for every chunk the forward issued 10 vector instructions per
// score, with this 7.)  A thread's chunks lie RS rows apart, a scalar step.
constexpr uint32_t NO_ROW = 0x80000000u;
template <class T, int DP, int ROWS, int NT> struct Stage {
  using L = Tile<T, DP>;
  static_assert(NT % L::CPR == 0 && (ROWS * L::CPR < NT || ROWS * L::CPR % NT == 0), "whole rows per turn");
  static constexpr int CH = ROWS * L::CPR;
  static constexpr int NI = (CH + NT - 1) / NT;
  static constexpr int RS = NT / L::CPR;              // rows between a thread's chunks
  u4 v[NI];
  uint32_t off;
  int step;
  // bytes(r): row r's distance from the tile's first row
  template <class Bytes> __device__ __forceinline__ void init(int D, Bytes bytes) {
    const int r = threadIdx.x / L::CPR, c = threadIdx.x % L::CPR;
    off = (CH < NT && (int)threadIdx.x >= CH) || c * L::EPC >= D ? NO_ROW : bytes(r) + 16 * c;
    step = (int)bytes(RS);
  }
  // rows 0 .. left - 1 from `first` (uniform over the workgroup)
  __device__ __forceinline__ void load(const T* first, int left) {
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(first), 0, 0x7fffffff, 0x00020000);
    const int r = threadIdx.x / L::CPR;
    // (one load for whole and partial tiles: two alternatives would be merged behind a wait)
#pragma unroll
    for (int i = 0; i < NI; ++i)
      v[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, r < left - i * RS ? off : NO_ROW, i * step, 0);
  }
  __device__ __forceinline__ void store(char* s) const {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int id = threadIdx.x + i * NT;
      if (CH < NT && id >= CH) continue;
      *reinterpret_cast<u4*>(s + L::at(id / L::CPR, id % L::CPR)) = v[i];
    }
  }
};
// The operands loaded before a main loop have arrived: said once here, or the compiler's counts, merged
// over the loop's entries, wait for the prefetched tile before each first product.
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }   // vmcnt(0)

template <int N> struct Int { static constexpr int value = N; };

// Orders the LDS reads of the N fragment products before it: AHEAD fragments (PER reads each) are in
// flight before the first product, then each product (MUL of them a fragment) is followed by the next fragment's reads.
// (Left to itself the compiler reads, waits and multiplies one fragment at a time.)
template <int N, int PER, int AHEAD, int MUL = 1> __device__ __forceinline__ void feed() {
  constexpr int A = AHEAD < N ? AHEAD : N;
  __builtin_amdgcn_sched_group_barrier(0x100, A * PER, 0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, MUL, 0);
    if (i + A < N) __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
  }
}

__device__ __forceinline__ float load_f32(const float* base, uint32_t off) {   // base uniform; NO_ROW: 0
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), 0, 0x7fffffff, 0x00020000);
  return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rsrc, off, 0, 0));
}

// a lane's fragments of one row, `off` bytes from `base` (uniform); NO_ROW: zeros
template <class T, int DP> using Frags = typename Ty<T>::Frag[Tile<T, DP>::NCH];
template <class T, int DP>
__device__ __forceinline__ void load_frags(Frags<T, DP>& f, const T* base, uint32_t off, int D, int h) {
  using L = Tile<T, DP>;
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, 0x7fffffff, 0x00020000);
#pragma unroll
  for (int k = 0; k < L::NCH; ++k) {
    const int d = k * L::KC + h * L::EPC;
    f[k] = __builtin_bit_cast(typename Ty<T>::Frag,
                              __builtin_amdgcn_raw_buffer_load_b128(rsrc, d < D ? off + d * (uint32_t)sizeof(T) : NO_ROW, 0, 0));
  }
}

// one column's accumulators (rows = features), scaled, to D consecutive elements
template <class U, int DT>
__device__ __forceinline__ void store_col(U* p, const f16v (&o)[DT], float f, int D, int h) {
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 32 * dt + 8 * q + 4 * h;
      if (d < D) {
        const f4 x = {o[dt][4 * q] * f, o[dt][4 * q + 1] * f, o[dt][4 * q + 2] * f, o[dt][4 * q + 3] * f};
        *reinterpret_cast<typename Ty<U>::Quad*>(p + d) = __builtin_convertvector(x, typename Ty<U>::Quad);
      }
    }
}

// The bias of every relative position for one head, log2 domain: -R .. R and MARGIN more on either
// side that repeat the ends, so that a tile which is not wholly beyond +-R reads without clamping.
// A bias below LOWEST (log2 domain, -11356 in the table) masks, as -inf does: fp32 statistics could not hold the score beside it.
constexpr int MARGIN = 64, SKEW = 2048;
constexpr float LOWEST = -16384.f;
__host__ __device__ __forceinline__ int span_of(int R) { return 2 * (R + MARGIN) + 1; }
template <class T, int NT>
__device__ __forceinline__ void load_bias(const Args& a, float* lut, int head) {
  const T* tb = reinterpret_cast<const T*>(a.p.table);
  const int R = a.p.max_distance;
  for (int i = threadIdx.x; i < span_of(R); i += NT) {
    const int b = min(max(a.p.lut[min(max(i - MARGIN, 0), 2 * R)], 0), a.p.num_buckets - 1);
    const float x = (float)tb[(int64_t)b * a.p.Hq + head] * LOG2E;
    lut[i] = x < LOWEST ? -INF : x;
  }
}

__device__ __forceinline__ int acc_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// the LDS accesses of this wave's lanes before and after stay in program order: the hardware keeps it within
// a wave, this holds the compiler to it where lanes read what other lanes wrote (no instruction)
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
}

// a value that is the same in every lane, told to the compiler (scalar registers and branches)
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A row of a tile table, held to the packed tensors: whatever a table that was overwritten or freed says, no access
// leaves them (scalar operations, ten a workgroup).
struct Where {
  int q0, k0, nq, nk, first;
  __device__ __forceinline__ Where(const Args& a, const int32_t* t, bool queries) {
    auto in = [&](int i, int most) { return min(max(uni(t[i]), 0), most); };
    const int Tq = (int)a.p.total_q, Tk = (int)a.p.total_k;
    q0 = in(0, Tq);
    k0 = in(1, Tk);
    nq = in(2, min(Tq - q0, a.p.max_q));
    nk = in(3, min(Tk - k0, a.p.max_k));
    first = in(4, queries ? nq : nk);
  }
};

// where a workgroup's query tile lies
struct QTile {
  int pos0, nq, nk, npos, nrows, off, kvh, head0;
  int64_t q0, k0;
  __device__ __forceinline__ QTile(const Args& a, int tile, int hidx) {
    const Where at(a, a.p.q_tiles + 8 * (int64_t)tile, true);
    q0 = at.q0;
    k0 = at.k0;
    nq = at.nq;
    nk = at.nk;
    pos0 = at.first;
    off = nk - nq;
    npos = min(a.p.q_tile, nq - pos0);
    nrows = npos * a.pg;
    kvh = hidx / a.nsub;
    head0 = kvh * a.group + (hidx - kvh * a.nsub) * a.pg;
  }
  __device__ __forceinline__ int limit(const Args& a, int row) const {   // keys that row sees
    return a.p.causal ? min(max(pos0 + div_pg(a, row) + off + 1, 0), nk) : nk;
  }
};

// scores of one 32x32 tile to the log2 domain with bias, s c + bias + more.  Register r's relative position is
// rel0 + SIGN acc_row(r, h); lo .. hi (uniform) bounds those of the tile.
template <int SIGN, bool MORE>
__device__ __forceinline__ void add_bias(f16v& s, float c, const float* lut, int rel0, int lo, int hi, int h, int R,
                                         float more = 0.f) {
  if (hi <= -R || lo >= R) {                               // one bucket for the whole tile
    const float b = lut[hi <= -R ? 0 : 2 * (R + MARGIN)] + more;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c, b);
  } else {
    const float* p = lut + (rel0 + SIGN * 4 * h + R + MARGIN);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c, MORE ? p[SIGN * acc_row(r, 0)] + more : p[SIGN * acc_row(r, 0)]);
  }
}

// -------------------------------------------------------------------------------------------
// forward
// -------------------------------------------------------------------------------------------
// keys of a tile.  32 in two-wave workgroups at head_dim 128: few rows are bound by the reads of K and V, and
// 32 KB of LDS let four of them run on a CU (one token over 32 caches of up to 16384 keys, 0.43 GB: 64 keys 124 us, 32 96 us).
template <class T, int DP, int NW> constexpr int key_tile() { return sizeof(T) == 4 || (DP == 128 && NW == 2) ? 32 : 64; }
// dK / dV at head_dim 128 hold 128 registers of sums: V goes to LDS and the row tile is 32, so that two
// waves per SIMD fit (causal training step of 10 k tokens, 16 heads over 4: V in registers at one
// wave 0.59 ms, at two, spilling, 1.50 ms; so 0.50 ms)
template <class T, int DP> constexpr bool v_in_lds() { return sizeof(T) == 2 && DP == 128; }
// waves per SIMD the registers are budgeted for.  One (all 512 registers) where two would spill: fp32 at
// wide heads, and in the backward two-wave workgroups and a bias at head_dim 128.  Four in the 16-bit forward at
// head_dim 64: its vector work per score is the bound, and waves of four workgroups fill each other's waits
// (sequences of 300 to 982 with a bias, 16 heads, bf16: two 99 us, three 98, four, with 5 registers spilled before the loop, 90).
template <class T, int DP, int NW> constexpr int occ_fwd() {
  return DP == 128 && sizeof(T) == 4 ? 1 : DP == 64 && sizeof(T) == 2 && NW == 4 ? 4 : 2;
}
template <class T, int DP, bool BIAS, int NW> constexpr int occ_bwd() {
  return (sizeof(T) == 4 && DP >= 64) || (DP == 128 && (NW == 2 || BIAS)) ? 1 : 2;
}
// query rows of a tile in dK / dV
template <class T, int DP> constexpr int row_tile() { return sizeof(T) == 4 || v_in_lds<T, DP>() ? 32 : 64; }

template <class T, int DP, bool BIAS, int NW>
__global__ __launch_bounds__(NW * 64, (occ_fwd<T, DP, NW>())) void fwd_kernel(Args a) {
  using L = Tile<T, DP>;
  constexpr int NT = NW * 64, BN = key_tile<T, DP, NW>(), NB = BN / 32, TILE = BN * L::RB;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* lut = reinterpret_cast<float*>(smem + 4 * TILE);
  const int nh = a.p.Hkv * a.nsub;
  const int hidx = blockIdx.x % nh;
  const QTile t(a, blockIdx.x / nh, hidx);
  const int lane = threadIdx.x & 63, w = uni(threadIdx.x >> 6), h = lane >> 5, D = a.p.D, R = a.p.max_distance;
  const int row = w * 32 + (lane & 31), dpos = div_pg(a, row);
  const bool valid = row < t.nrows;
  const int head = t.head0 + row - dpos * a.pg;
  const int qfirst = t.pos0 + w * 32 + t.off, qabs = t.pos0 + dpos + t.off;   // (a bias: one head per tile, row = position)
  const bool active = w * 32 < t.nrows;
  const int wmin = uni(t.limit(a, w * 32)), wmax = active ? uni(t.limit(a, min(w * 32 + 31, t.nrows - 1))) : 0;
  const int kend = t.nrows > 0 ? uni(t.limit(a, t.nrows - 1)) : 0;
  const int nt = (kend + BN - 1) / BN, t0 = blockIdx.y * a.per_q, t1 = min(nt, t0 + a.per_q);

  f16v o[L::DT];
#pragma unroll
  for (int i = 0; i < L::DT; ++i) o[i] = f16v{};
  // the origin (0 until a key is seen) and the largest score beside it that leaves it where it is.  Behind keys that
  // score far below (a bias puts them there), the origin is far below too, and a score on top of it would lose its
  // digits: DEPTH of it at most are taken off at once (2^-18 of P), the rest once the tile's own largest score is known.
  constexpr float BELOW = __is_same(T, _Float16) ? 7.f : 0.f, ROOM = __is_same(T, _Float16) ? 15.f : 8.f, DEPTH = 64.f;
  float m = 0.f, most = -INF, l = 0.f;

  const T* kb = reinterpret_cast<const T*>(a.p.k) + t.k0 * a.p.k_ts + t.kvh * a.p.k_hs;
  const T* vb = reinterpret_cast<const T*>(a.p.v) + t.k0 * a.p.v_ts + t.kvh * a.p.v_hs;
  Stage<T, DP, BN, NT> ks, vs;
  ks.init(D, [&](int r) { return (uint32_t)r * (uint32_t)(a.p.k_ts * sizeof(T)); });
  vs.init(D, [&](int r) { return (uint32_t)r * (uint32_t)(a.p.v_ts * sizeof(T)); });
  auto fetch = [&](int j) {
    ks.load(kb + (int64_t)j * BN * a.p.k_ts, t.nk - j * BN);
    vs.load(vb + (int64_t)j * BN * a.p.v_ts, t.nk - j * BN);
  };
  // every load of the prologue is in flight before the first wait
  if (t0 < t1) fetch(t0);
  typename Ty<T>::Frag qf[L::NCH];
  load_frags<T, DP>(qf, reinterpret_cast<const T*>(a.p.q) + (t.q0 + t.pos0) * a.p.q_ts + t.head0 * a.p.q_hs,
                    valid ? (uint32_t)((dpos * a.p.q_ts + (head - t.head0) * a.p.q_hs) * (int)sizeof(T)) : NO_ROW, D, h);
  if (BIAS) load_bias<T, NT>(a, lut, t.head0);
  if (t0 < t1) {
    ks.store(smem);
    vs.store(smem + TILE);
  }
  loads_done();
  __syncthreads();
  typename L::Lane at(lane);
  auto step = [&](int j, auto buf) {
    at.renew();
    const char* K = smem + buf.value * 2 * TILE;
    const char* V = K + TILE;
    if (j + 1 < t1) fetch(j + 1);
    const int base = j * BN;
    if (base < wmax) {
      f16v s[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        s[n] = f16v{};
#pragma unroll
        for (int k = 0; k < L::NCH; ++k) s[n] = mma(L::row(K, at, 32 * n, k), qf[k], s[n]);
      }
      feed<NB * L::NCH, 1, 4>();
      // to the log2 domain, from the running origin m on: s c [+ bias] - m
      const float from = fminf(-m, DEPTH);
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        if constexpr (BIAS) {
          add_bias<1, true>(s[n], a.c, lut, base + 32 * n - qabs, base + 32 * n - qfirst - 31, base + 32 * n - qfirst + 31, h, R, from);
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) s[n][r] = fmaf(s[n][r], a.c, from);
        }
      }
      if (base + BN > wmin) {
        // (found again from the lane's number: it would take a register through the loop)
        uint32_t all = ~0u;
        asm volatile("" : "+v"(all));
        const int lim = t.limit(a, w * 32 + (int)(__builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0u)) & 31));
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (base + 32 * n + acc_row(r, h) >= lim) s[n][r] = -INF;
      }
      float mt = s[0][0];
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[n][r]);
      mt = xmax32(mt);
      // the origin moves when the first key is seen, and only when a score exceeds it by 2^8 after that:
      // exp2 stays <= 2^8, the sums are fp32.  fp16: it lies 2^7 below the largest score and moves at 2^15, so that P
      // is a normal number down to 2^-21 of the largest (with the origin at the largest, down to 2^-14: 131072 keys
      // 2^-17 below one took o 0.18 percent off)
      if (__builtin_amdgcn_ballot_w64(mt > most) != 0) {
        const bool first = most == -INF && !(-m > DEPTH);
        mt += -m - from;
        const float up = first ? mt - BELOW : fmaxf(mt - BELOW, 0.f), old = m;
        const bool none = up == -INF;
        m = none ? 0.f : m + up;
        const float f = first ? 0.f : __builtin_amdgcn_exp2f(old - m);   // (sums and scores move as far as m did, rounded)
        const float by = none ? 0.f : m + from;
        most = none || -m > DEPTH ? -INF : ROOM;
        l *= f;
#pragma unroll
        for (int i = 0; i < L::DT; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[i][r] *= f;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[n][r] -= by;
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[n][r] = __builtin_amdgcn_exp2f(s[n][r]);
#pragma unroll
        for (int r = 0; r < 16; r += 4) l += (s[n][r] + s[n][r + 1]) + (s[n][r + 2] + s[n][r + 3]);
      }
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int b = 0; b < L::TB; ++b) {
          const auto pf = take<T>(s[n], b);
#pragma unroll
          for (int dt = 0; dt < L::DT; ++dt) o[dt] = mma(L::col(V, at, 32 * n, b, dt), pf, o[dt]);
        }
      // (with a bias and 128 registers, three fragments ahead do not fit and each is waited for: 91.2 us for the sequences
      // of 300 to 982 above, two 90.5)
      feed<NB * L::TB * L::DT, L::CR, BIAS && occ_fwd<T, DP, NW>() == 4 ? 2 : 3>();
    }
    if (j + 1 < t1) {
      char* Kn = smem + (1 - buf.value) * 2 * TILE;
      ks.store(Kn);
      vs.store(Kn + TILE);
    }
    __syncthreads();
  };
  for (int j = t0; j < t1; j += 2) {
    step(j, Int<0>{});
    if (j + 1 < t1) step(j + 1, Int<1>{});
  }
  l = xsum32(l);
  if (!valid) return;
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);      // (a NaN sum stays one)
  const float lse = l == 0.f ? INF : m + __log2f(l);
  const int64_t rid = (t.q0 + t.pos0 + dpos) * a.p.Hq + head;
  if (a.split_q == 1) {
    store_col(reinterpret_cast<T*>(a.p.o) + rid * D, o, inv, D, h);
    if (h == 0) a.p.lse[rid] = lse;
  } else {
    const int64_t pid = (int64_t)blockIdx.y * a.p.total_q * a.p.Hq + rid;
    if (t0 < t1) store_col(a.part + pid * D, o, inv, D, h);    // (the join reads no part that saw nothing)
    if (h == 0) a.part_lse[pid] = lse;
  }
}

// Joins the n <= 64 parts of `rows` rows of D: weighted by their log-sum-exp (WEIGHTED: the forward; +inf
// marks a part that saw nothing and was not written) or plainly summed, in the order of the parts.  8 rows per
// workgroup, 32 lanes of 4 columns each; a lane takes the weights of parts l and l + 32, and eight parts
// are in flight (one after the other: 12 us instead of 5 for 20 parts of 1024 rows).
template <class T, bool WEIGHTED>
__global__ __launch_bounds__(256) void join_kernel(const float* part, const float* part_lse, int n, int64_t rows,
                                                   int D, T* out, T* out2, float* lse) {
  if (blockIdx.y == 1) {                               // (the second tensor's parts follow the first's)
    part += (int64_t)n * rows * D;
    out = out2;
  }
  const int l = threadIdx.x & 31, d = l * 4;
  const int64_t row0 = (int64_t)blockIdx.x * 8, row = row0 + (threadIdx.x >> 5);
  const bool live = row < rows;
  float w[2] = {l < n ? 1.f : 0.f, l + 32 < n ? 1.f : 0.f};
  if (WEIGHTED) {
    float x[2] = {INF, INF};
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (live && l + 32 * i < n) x[i] = part_lse[(int64_t)(l + 32 * i) * rows + row];
#pragma unroll
    for (int i = 0; i < 2; ++i) if (x[i] == INF) x[i] = -INF;
    float m = fmaxf(x[0], x[1]);                       // (a NaN is not lost: its weight below is one)
    m = xmax16(m);
    m = fmaxf(m, dpp_mov<0x128>(m));
    m = fmaxf(m, dpp_mov<0x124>(m));
    m = fmaxf(m, dpp_mov<0x4e>(m));
    m = fmaxf(m, dpp_mov<0xb1>(m));
#pragma unroll
    for (int i = 0; i < 2; ++i) w[i] = x[i] == -INF ? 0.f : __builtin_amdgcn_exp2f(x[i] - m);
    float sum = w[0] + w[1];
    sum = xsum16(sum);
    sum += dpp_mov<0x128>(sum);
    sum += dpp_mov<0x124>(sum);
    sum += dpp_mov<0x4e>(sum);
    sum += dpp_mov<0xb1>(sum);
#pragma unroll
    for (int i = 0; i < 2; ++i) w[i] = w[i] == 0.f ? 0.f : w[i] / sum;
    if (live && l == 0) lse[row] = sum == 0.f ? INF : m + __log2f(sum);
  }
  f4 acc = {0.f, 0.f, 0.f, 0.f};
  const uint32_t at = live && d < D ? (uint32_t)(((threadIdx.x >> 5) * D + d) * 4) : NO_ROW;
  for (int i0 = 0; i0 < n; i0 += 8) {
    f4 p[8];
    float wi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      wi[i] = __shfl(i0 < 32 ? w[0] : w[1], (i0 + i) & 31, 32);
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(part + ((int64_t)min(i0 + i, n - 1) * rows + row0) * D),
                                                          0, 0x7fffffff, 0x00020000);
      p[i] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, wi[i] != 0.f ? at : NO_ROW, 0, 0));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(wi[i], p[i][e], acc[e]);
  }
  if (live && d < D) *reinterpret_cast<typename Ty<T>::Quad*>(out + row * D + d) = __builtin_convertvector(acc, typename Ty<T>::Quad);
}

// -------------------------------------------------------------------------------------------
// backward: dQ (and rowsum(dO O), the bias sums by relative position)
// -------------------------------------------------------------------------------------------
// fp16 has few exponents, so its dS enters the products times a power of two that is taken out of the fp32
// results.  Each column (a query's dQ, a key's dK) has its own, from the largest |dS| it has met: that one
// lies in [2^12, 2^13) when the power is chosen, and a larger one may come up to 2^15 before the power is
// chosen again and the sums so far are scaled to it (exact; a tile or two of a walk).  Nothing of another row,
// sequence or batch enters, no size of dO or v overflows, and of the second part 2^-37 of the column's largest dS is
// lost at most, however many keys share the row.  (One power for a whole batch from max |dO|, with room for |v| of 2^18,
// left nothing of the second part from 65536 keys on, or beside a sequence of larger gradients.)
// bf16 and fp32 have fp32's range and take 1.  Measured, training with 12 heads of 64: 113 us for the launch with the
// batch's power, 121 so, without the launch of 2.4 us that found max |dO|.
struct Power {
  float up = 1.f, down = 1.f, most = 0x1p-100f;   // 1 / the power, the power, the |dS| up to which it stays (below 2^-100: nothing)
  // chosen again for this lane's largest |dS|: what the sums so far are multiplied by
  __device__ __forceinline__ float choose(float big) {
    if (!(big > most)) return 1.f;
    const uint32_t e = min(__float_as_uint(big) >> 23, 254u);      // (an infinity: its column is lost anyway)
    const float p = __uint_as_float(e << 23), old = up;
    up = p * 0x1p-12f;
    down = 1.f / up;
    most = p * 8.f;
    return old * down;
  }
};
// one 32 x 32 tile of dS in fp32 -> times its columns' powers; acc: the sums so far
template <int DT> __device__ __forceinline__ void fit(f16v& ds, Power& pw, f16v (&acc)[DT]) {
  float big = fabsf(ds[0]);
#pragma unroll
  for (int r = 1; r < 16; ++r) big = fmaxf(big, fabsf(ds[r]));
  if (__builtin_amdgcn_ballot_w64(big > pw.most) != 0) {
    const float f = pw.choose(xmax32(big));        // (lanes l and l ^ 32 share a column)
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][r] *= f;
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) ds[r] *= pw.down;
}

// acc += X^T dS over the rows of contraction block t.  fp16's dS goes in two parts: rounded once it would be off
// as much as the gradient's own rounding (1.5 roundings in all, so 1.1), and fp16 is chosen for its
// digits (training, 12 heads of 64: the launch 102 -> 112 us, before the powers).  bf16 keeps one part
// (10 k tokens, 16 heads of 128 over 4: two would take 910 us instead of 765).
template <class L, class Lane> __device__ __forceinline__ void add_ds(f16v (&acc)[L::DT], const char* x, const Lane& at, int row0, int t, const f16v& ds) {
  using T = typename L::Type;
  const auto whole = take<T>(ds, t);
  if constexpr (__is_same(T, _Float16)) {
    const auto rest = rest_of<T>(ds, t, whole);
#pragma unroll
    for (int dt = 0; dt < L::DT; ++dt) {
      const auto xt = L::col(x, at, row0, t, dt);
      acc[dt] = mma(xt, whole, acc[dt]);
      acc[dt] = mma(xt, rest, acc[dt]);
    }
  } else {
#pragma unroll
    for (int dt = 0; dt < L::DT; ++dt) acc[dt] = mma(L::col(x, at, row0, t, dt), whole, acc[dt]);
  }
}

template <class T, int DP, bool BIAS, int NW>
__device__ __forceinline__ void dq_body(const Args& a, int wg, int part_no) {
  using L = Tile<T, DP>;
  constexpr int NT = NW * 64, BN = key_tile<T, DP, NW>(), NB = BN / 32, TILE = BN * L::RB;
  constexpr bool HALF = __is_same(T, _Float16);
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int nsplit = a.split_q;
  const int R = a.p.max_distance, NH = 2 * R + 1;
  float* lut = reinterpret_cast<float*>(smem + 4 * TILE);
  float* hist = lut + span_of(R) * (1 + (threadIdx.x >> 6));   // this wave's sums by relative position
  float* skew = lut + (span_of(R) * (1 + NW) + 3) / 4 * 4 + SKEW * (threadIdx.x >> 6);   // and 32 x 64 to take them
  const int nh = a.p.Hkv * a.nsub;
  const int hidx = wg % nh;
  const QTile t(a, wg / nh, hidx);
  const int lane = threadIdx.x & 63, w = uni(threadIdx.x >> 6), h = lane >> 5, D = a.p.D;
  const bool sums = BIAS && a.p.dtable != nullptr;

  const int row = w * 32 + (lane & 31), dpos = div_pg(a, row);
  const bool valid = row < t.nrows;
  const int head = t.head0 + row - dpos * a.pg;
  const int lim = valid ? t.limit(a, row) : 0;
  const int qfirst = t.pos0 + w * 32 + t.off, qabs = t.pos0 + dpos + t.off;   // (a bias: one head per tile, row = position)
  const bool active = w * 32 < t.nrows;
  const int wmin = w * 32 + 31 < t.nrows ? uni(t.limit(a, w * 32)) : 0;
  const int wmax = active ? uni(t.limit(a, min(w * 32 + 31, t.nrows - 1))) : 0;
  const int kend = t.nrows > 0 ? uni(t.limit(a, t.nrows - 1)) : 0;
  const int nt = (kend + BN - 1) / BN, t0 = part_no * a.per_q, t1 = min(nt, t0 + a.per_q);

  const T* kb = reinterpret_cast<const T*>(a.p.k) + t.k0 * a.p.k_ts + t.kvh * a.p.k_hs;
  const T* vb = reinterpret_cast<const T*>(a.p.v) + t.k0 * a.p.v_ts + t.kvh * a.p.v_hs;
  Stage<T, DP, BN, NT> ks, vs;
  ks.init(D, [&](int r) { return (uint32_t)r * (uint32_t)(a.p.k_ts * sizeof(T)); });
  vs.init(D, [&](int r) { return (uint32_t)r * (uint32_t)(a.p.v_ts * sizeof(T)); });
  auto fetch = [&](int j) {
    ks.load(kb + (int64_t)j * BN * a.p.k_ts, t.nk - j * BN);
    vs.load(vb + (int64_t)j * BN * a.p.v_ts, t.nk - j * BN);
  };
  if (t0 < t1) fetch(t0);
  const int64_t tok0 = t.q0 + t.pos0, rid0 = tok0 * a.p.Hq + t.head0;
  const int rofs = dpos * a.p.Hq + head - t.head0;
  const int64_t rid = rid0 + rofs;
  typename Ty<T>::Frag qf[L::NCH], gf[L::NCH];
  load_frags<T, DP>(qf, reinterpret_cast<const T*>(a.p.q) + tok0 * a.p.q_ts + t.head0 * a.p.q_hs,
                    valid ? (uint32_t)((dpos * a.p.q_ts + (head - t.head0) * a.p.q_hs) * (int)sizeof(T)) : NO_ROW, D, h);
  load_frags<T, DP>(gf, reinterpret_cast<const T*>(a.p.dout) + tok0 * a.p.do_ts + t.head0 * a.p.do_hs,
                    valid ? (uint32_t)((dpos * a.p.do_ts + (head - t.head0) * a.p.do_hs) * (int)sizeof(T)) : NO_ROW, D, h);
  const float lse_in = load_f32(a.p.lse + rid0, valid ? 4u * rofs : NO_ROW);
  const float delta = load_f32(a.delta + rid0, valid ? 4u * rofs : NO_ROW);
  if (BIAS) load_bias<T, NT>(a, lut, t.head0);
  if (sums) {
    for (int i = lane; i < span_of(R); i += 64) hist[i] = 0.f;
    for (int i = lane; i < SKEW; i += 64) skew[i] = 0.f;
  }
  const float lse = valid ? lse_in : INF;
  Power power;
  // dP starts from -delta where the registers allow a copy of it (one subtraction less per score)
  constexpr bool FROM = DP <= 64;
  f16v minus;
#pragma unroll
  for (int r = 0; r < 16; ++r) minus[r] = FROM ? -delta : 0.f;

  f16v o[L::DT];
#pragma unroll
  for (int i = 0; i < L::DT; ++i) o[i] = f16v{};
  float far_lo = 0.f, far_hi = 0.f;
  if (t0 < t1) {
    ks.store(smem);
    vs.store(smem + TILE);
  }
  loads_done();
  __syncthreads();
  typename L::Lane at(lane);
  auto step = [&](int j, auto buf) {
    at.renew();
    const char* K = smem + buf.value * 2 * TILE;
    const char* V = K + TILE;
    if (j + 1 < t1) fetch(j + 1);
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int base = j * BN + 32 * n;
      if (base < wmax) {
        f16v s = f16v{}, g = minus;
#pragma unroll
        for (int k = 0; k < L::NCH; ++k) s = mma(L::row(K, at, 32 * n, k), qf[k], s);
#pragma unroll
        for (int k = 0; k < L::NCH; ++k) g = mma(L::row(V, at, 32 * n, k), gf[k], g);
        feed<2 * L::NCH, 1, 4>();
        const float c = BIAS ? 1.f : a.c;
        const int rel0 = base - qabs;
        const int lo = base - qfirst - 31, hi = base - qfirst + 31;   // the tile's relative positions
        if (BIAS) add_bias<1, true>(s, a.c, lut, rel0, lo, hi, h, R, -lse);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, BIAS ? 0.f : -lse)) * (FROM ? g[r] : g[r] - delta);
        if (base + 32 > wmin) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (base + acc_row(r, h) >= lim) s[r] = 0.f;
        }
        if (sums) {
          if (hi <= -R) {
#pragma unroll
            for (int r = 0; r < 16; ++r) far_lo += s[r];
          } else if (lo >= R) {
#pragma unroll
            for (int r = 0; r < 16; ++r) far_hi += s[r];
          } else {
            // Row i's keys are written i places further left, so that a column holds one distance: lane d
            // sums column d over the 32 rows and adds it to this wave's sums.  (Places that no key
            // reaches stay zero.  Adding each score atomically took 280 cycles for 32 of them: dQ 145 us
            // instead of 81, fp16 training with 12 heads of 64.)
            float* p = skew + 63 * (lane & 31) + 4 * h + 31;
#pragma unroll
            for (int r = 0; r < 16; ++r) p[acc_row(r, 0)] = s[r];
            wave_order();
            float x = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) x += skew[64 * i + lane];
            // column d: distance base - qfirst + d - 31; column 63 holds nothing
            float* q = hist + (lo + lane + R + MARGIN);
            *q += x;
            wave_order();                                      // (the next tile writes the rows and adds to these sums)
          }
        }
        if (HALF) fit(s, power, o);
#pragma unroll
        for (int b = 0; b < L::TB; ++b) {
          add_ds<L>(o, K, at, 32 * n, b, s);
        }
        feed<L::TB * L::DT, L::CR, 3, HALF ? 2 : 1>();
      }
    }
    if (j + 1 < t1) {
      char* Kn = smem + (1 - buf.value) * 2 * TILE;
      ks.store(Kn);
      vs.store(Kn + TILE);
    }
    __syncthreads();
  };
  for (int j = t0; j < t1; j += 2) {
    step(j, Int<0>{});
    if (j + 1 < t1) step(j + 1, Int<1>{});
  }
  if (sums) {
    // the margins belong to the two ends
    for (int i = lane; i <= MARGIN; i += 64) {
      far_lo += hist[i];
      far_hi += hist[2 * R + MARGIN + i];
    }
    far_lo = wave_sum(far_lo);
    far_hi = wave_sum(far_hi);
    wave_order();
    if (lane == 0) {
      hist[MARGIN] = far_lo;
      hist[2 * R + MARGIN] = far_hi;                           // (R >= 1: not the same place)
    }
    __syncthreads();
    float* out = a.hist + ((int64_t)part_no * a.wgs_q + wg) * NH;
    for (int i = threadIdx.x; i < NH; i += NT) {
      float x = 0.f;
#pragma unroll
      for (int v = 0; v < NW; ++v) x += lut[(1 + v) * span_of(R) + MARGIN + i];
      out[i] = x;
    }
  }
  if (!valid) return;
  const float f = a.p.scale * power.up;
  if (nsplit == 1) store_col(reinterpret_cast<T*>(a.p.dq) + rid * D, o, f, D, h);
  else store_col(a.part + ((int64_t)part_no * a.p.total_q * a.p.Hq + rid) * D, o, f, D, h);
}

// delta from P and dP themselves, rowsum(P dP), which makes a row's dS sum to zero: for the bias table's gradient in bf16.  A
// bucket of nearly all keys gets the small rest of a row's terms, and the error of rowsum(dO O), from the roundings
// of O and of the forward's P, stays whole in it: 0.8 to 2.2 % of the table's gradient with 5 queries over 9001 keys, with
// this 0.2 %, the output's own rounding.  (fp16's roundings are eight times smaller: it keeps delta_kernel.)  Two
// products of dQ's walk and one sum a row, the keys in parts, which add_parts_kernel adds: training with 12 heads of
// 64, up to 2047 tokens, 38 us instead of delta_kernel's 6 beside 97 us of bwd_kernel and 43 forward.
template <class T, int DP, int NW> constexpr int occ_row() { return DP == 128 ? 2 : NW == 4 ? 3 : 2; }
template <class T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, (occ_row<T, DP, NW>())) void row_kernel(Args a, float* out) {
  using L = Tile<T, DP>;
  constexpr int NT = NW * 64, BN = key_tile<T, DP, NW>(), NB = BN / 32, TILE = BN * L::RB;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* lut = reinterpret_cast<float*>(smem + 4 * TILE);
  const int nh = a.p.Hkv * a.nsub, hidx = blockIdx.x % nh, R = a.p.max_distance, D = a.p.D;
  const QTile t(a, blockIdx.x / nh, hidx);
  const int lane = threadIdx.x & 63, w = uni(threadIdx.x >> 6), h = lane >> 5, row = w * 32 + (lane & 31);   // (one head per tile)
  const bool valid = row < t.nrows;
  const int lim = valid ? t.limit(a, row) : 0;
  const int qfirst = t.pos0 + w * 32 + t.off;
  const int wmin = w * 32 + 31 < t.nrows ? uni(t.limit(a, w * 32)) : 0;
  const int wmax = w * 32 < t.nrows ? uni(t.limit(a, min(w * 32 + 31, t.nrows - 1))) : 0;
  const int kend = t.nrows > 0 ? uni(t.limit(a, t.nrows - 1)) : 0;
  const int nt = (kend + BN - 1) / BN, t0 = blockIdx.y * a.per_r, t1 = min(nt, t0 + a.per_r);
  const int64_t tok0 = t.q0 + t.pos0, rid0 = tok0 * a.p.Hq + t.head0;
  out += (int64_t)blockIdx.y * a.p.total_q * a.p.Hq + rid0 + row * a.p.Hq;
  if (t0 >= t1) {                                      // (the whole workgroup)
    if (valid && h == 0) *out = 0.f;
    return;
  }
  const T* kb = reinterpret_cast<const T*>(a.p.k) + t.k0 * a.p.k_ts + t.kvh * a.p.k_hs;
  const T* vb = reinterpret_cast<const T*>(a.p.v) + t.k0 * a.p.v_ts + t.kvh * a.p.v_hs;
  Stage<T, DP, BN, NT> ks, vs;
  ks.init(D, [&](int r) { return (uint32_t)r * (uint32_t)(a.p.k_ts * sizeof(T)); });
  vs.init(D, [&](int r) { return (uint32_t)r * (uint32_t)(a.p.v_ts * sizeof(T)); });
  auto fetch = [&](int j) {
    ks.load(kb + (int64_t)j * BN * a.p.k_ts, t.nk - j * BN);
    vs.load(vb + (int64_t)j * BN * a.p.v_ts, t.nk - j * BN);
  };
  fetch(t0);
  typename Ty<T>::Frag qf[L::NCH], gf[L::NCH];
  load_frags<T, DP>(qf, reinterpret_cast<const T*>(a.p.q) + tok0 * a.p.q_ts + t.head0 * a.p.q_hs,
                    valid ? (uint32_t)(row * a.p.q_ts * (int)sizeof(T)) : NO_ROW, D, h);
  load_frags<T, DP>(gf, reinterpret_cast<const T*>(a.p.dout) + tok0 * a.p.do_ts + t.head0 * a.p.do_hs,
                    valid ? (uint32_t)(row * a.p.do_ts * (int)sizeof(T)) : NO_ROW, D, h);
  const float lse_in = load_f32(a.p.lse + rid0, valid ? 4u * (row * a.p.Hq) : NO_ROW);
  load_bias<T, NT>(a, lut, t.head0);
  const float lse = valid ? lse_in : INF;
  float sum = 0.f;
  ks.store(smem);
  vs.store(smem + TILE);
  loads_done();
  __syncthreads();
  typename L::Lane at(lane);
  auto step = [&](int j, auto buf) {
    at.renew();
    const char* K = smem + buf.value * 2 * TILE;
    const char* V = K + TILE;
    if (j + 1 < t1) fetch(j + 1);
    if (j * BN < wmax) {
      f16v s[NB], g[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n) s[n] = g[n] = f16v{};
#pragma unroll
      for (int k = 0; k < L::NCH; ++k)
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          s[n] = mma(L::row(K, at, 32 * n, k), qf[k], s[n]);
          g[n] = mma(L::row(V, at, 32 * n, k), gf[k], g[n]);
        }
      feed<2 * NB * L::NCH, 1, 4>();
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const int base = j * BN + 32 * n;
        add_bias<1, true>(s[n], a.c, lut, base - qfirst - (lane & 31), base - qfirst - 31, base - qfirst + 31, h, R, -lse);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[n][r] = __builtin_amdgcn_exp2f(s[n][r]) * g[n][r];
        if (base + 32 > wmin) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (base + acc_row(r, h) >= lim) s[n][r] = 0.f;
        }
#pragma unroll
        for (int r = 0; r < 16; r += 4) sum += (s[n][r] + s[n][r + 1]) + (s[n][r + 2] + s[n][r + 3]);
      }
    }
    if (j + 1 < t1) {
      char* Kn = smem + (1 - buf.value) * 2 * TILE;
      ks.store(Kn);
      vs.store(Kn + TILE);
    }
    __syncthreads();
  };
  for (int j = t0; j < t1; j += 2) {
    step(j, Int<0>{});
    if (j + 1 < t1) step(j + 1, Int<1>{});
  }
  sum = xsum32(sum);
  if (valid && h == 0) *out = sum;
}

// sums by relative position of the n workgroups of a head (workgroup i * Hq + head), 16 slices of
// them in order, then the slices in order: rel[head][NH]
__global__ __launch_bounds__(1024) void hist_sum_kernel(const float* hist, int n, int Hq, int NH, float* rel);
// dtable[b][head] = sum of rel[head][i] over the relative positions i of bucket b: a wave per bucket,
// each lane its positions in order, then the lanes (one thread per bucket took 15 us)
template <class T>
__global__ __launch_bounds__(1024) void hist_bucket_kernel(const float* rel, const int32_t* lut, int NH, int Hq, int nb,
                                                           T* dtable) {
  const int lane = threadIdx.x & 63;
  for (int b = threadIdx.x >> 6; b < nb; b += 16) {
    float x = 0.f;
    for (int i = lane; i < NH; i += 64) x += min(max(lut[i], 0), nb - 1) == b ? rel[(int64_t)blockIdx.x * NH + i] : 0.f;
    x = wave_sum(x);
    if (lane == 0) dtable[(int64_t)b * Hq + blockIdx.x] = (T)x;
  }
}

// -------------------------------------------------------------------------------------------
// backward: dK, dV
// -------------------------------------------------------------------------------------------
template <class T, int DP, bool BIAS, int NW>
__device__ __forceinline__ void dkv_body(const Args& a, int wg, int part_no) {
  using L = Tile<T, DP>;
  constexpr int NT = NW * 64, BQ = row_tile<T, DP>(), NB = BQ / 32, TILE = BQ * L::RB;
  constexpr bool VL = v_in_lds<T, DP>(), HALF = __is_same(T, _Float16);
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int nsplit = a.split_k;
  float* stat = reinterpret_cast<float*>(smem + 4 * TILE);     // [2][lse BQ | -delta BQ]
  float* lut = stat + 4 * BQ;
  char* vt = smem + 4 * TILE + 16 * BQ + (BIAS ? (span_of(a.p.max_distance) * 4 + 15) / 16 * 16 : 0);   // this tile's V (VL)
  const int kvh = wg % a.p.Hkv, tile = wg / a.p.Hkv, D = a.p.D, R = a.p.max_distance;
  const Where tl(a, a.p.k_tiles + 8 * (int64_t)tile, false);
  const int64_t q0 = tl.q0, k0 = tl.k0;
  const int nq = tl.nq, nk = tl.nk, key0 = tl.first, off = nk - nq;
  const int lane = threadIdx.x & 63, w = uni(threadIdx.x >> 6), h = lane >> 5;
  const int key = key0 + w * 32 + (lane & 31);
  const bool valid = key < nk;
  typename Ty<T>::Frag kf[L::NCH], vf[VL ? 1 : L::NCH];
  const int kr = w * 32 + (lane & 31);
  const T* vp = reinterpret_cast<const T*>(a.p.v) + (k0 + key0) * a.p.v_ts + kvh * a.p.v_hs;
  const uint32_t vofs = valid ? (uint32_t)(kr * a.p.v_ts * (int)sizeof(T)) : NO_ROW;
  load_frags<T, DP>(kf, reinterpret_cast<const T*>(a.p.k) + (k0 + key0) * a.p.k_ts + kvh * a.p.k_hs,
                    valid ? (uint32_t)(kr * a.p.k_ts * (int)sizeof(T)) : NO_ROW, D, h);
  if constexpr (VL) {
    typename Ty<T>::Frag f[L::NCH];                            // each wave writes and reads its own 32 rows
    load_frags<T, DP>(f, vp, vofs, D, h);
#pragma unroll
    for (int k = 0; k < L::NCH; ++k) *reinterpret_cast<typename Ty<T>::Frag*>(vt + L::at(w * 32 + (lane & 31), 2 * k + h)) = f[k];
  } else {
    load_frags<T, DP>(vf, vp, vofs, D, h);
  }
  f16v dk[L::DT], dv[L::DT];
#pragma unroll
  for (int i = 0; i < L::DT; ++i) dk[i] = dv[i] = f16v{};
  Power power;
  // fp16's P enters dV times 2^14 (at most 2^14 but for the rounding of scores: below 65504): over 16384 keys
  // and more P itself lies below the type's normal range (dV 10 roundings off at 200000 keys, so 1.4).  dS carries it too;
  // both are taken out at the end.
  constexpr float LIFT = HALF ? 14.f : 0.f, UNLIFT = HALF ? 0x1p-14f : 1.f;

  // rows (position * PK + head) that see any of the tile's keys, tile by tile, one head group after
  // the other: it = sub * ntq + row tile.  PK, the heads that share a row tile, is a power of two, so a
  // row tile holds whole positions and a thread's chunks lie whole positions apart.
  const int lg = a.pk_log, pk = 1 << lg, bp = BQ >> lg, nrows = nq << lg;
  const int first = a.p.causal ? min(max(key0 - off, 0), nq) / bp : 0;
  const int ntq = max((nq + bp - 1) / bp - first, 0), total = a.nsubk * ntq;
  const int t0 = part_no * a.per_k, t1 = min(total, t0 + a.per_k);
  // the first row that sees this lane's key / the wave's first and last key
  const int see = a.p.causal ? (key - off) * pk : 0;
  const int wfirst = a.p.causal ? (key0 + w * 32 - off) * pk : 0;
  const int wlast = a.p.causal ? (key0 + w * 32 + 31 - off) * pk : 0;
  const bool active = key0 + w * 32 < nk;

  Stage<T, DP, BQ, NT> qs, gs;
  float st_l, st_d;
  bool st_in;
  auto bytes = [&](int64_t ts, int64_t hs) {
    return [=](int r) { return (uint32_t)(((r >> lg) * ts + (r & (pk - 1)) * hs) * (int)sizeof(T)); };
  };
  qs.init(D, bytes(a.p.q_ts, a.p.q_hs));
  gs.init(D, bytes(a.p.do_ts, a.p.do_hs));
  const int sofs = ((int)threadIdx.x >> lg) * a.p.Hq + ((int)threadIdx.x & (pk - 1));
  auto fetch = [&](int it) {
    const int sub = it / ntq, pos = (first + it - sub * ntq) * bp, head0 = kvh * a.group + (sub << lg);
    const int left = min(nrows - (pos << lg), BQ);
    qs.load(reinterpret_cast<const T*>(a.p.q) + (q0 + pos) * a.p.q_ts + head0 * a.p.q_hs, left);
    gs.load(reinterpret_cast<const T*>(a.p.dout) + (q0 + pos) * a.p.do_ts + head0 * a.p.do_hs, left);
    const int64_t rid = (q0 + pos) * a.p.Hq + head0;
    const uint32_t at = (int)threadIdx.x < left ? 4u * sofs : NO_ROW;
    st_l = load_f32(a.p.lse + rid, at);
    st_d = load_f32(a.delta + rid, at);
    st_in = (int)threadIdx.x < left;
  };
  auto commit = [&](int b) {
    qs.store(smem + b * 2 * TILE);
    gs.store(smem + b * 2 * TILE + TILE);
    if (threadIdx.x < BQ) {
      stat[b * 2 * BQ + threadIdx.x] = st_in ? st_l - LIFT : INF;
      stat[b * 2 * BQ + BQ + threadIdx.x] = -st_d;
    }
  };
  int sub_now = -1;
  if (t0 < t1) {
    fetch(t0);
    commit(0);
  }
  loads_done();
  __syncthreads();
  typename L::Lane at(lane);
  auto step = [&](int it, auto buf) {
    at.renew();
    constexpr int b = buf.value;
    const char* Q = smem + b * 2 * TILE;
    const char* G = Q + TILE;
    const float* lse = stat + b * 2 * BQ;
    const float* dl = lse + BQ;
    const int sub = it / ntq, rb = (first + it - sub * ntq) * BQ;
    if (BIAS && sub != sub_now) {                              // the next head's biases
      __syncthreads();
      load_bias<T, NT>(a, lut, kvh * a.group + (sub << lg));
      __syncthreads();
      sub_now = sub;
    }
    if (it + 1 < t1) fetch(it + 1);
    if (active && rb + BQ > wfirst) {
      f16v s[NB], g[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        s[n] = f16v{};
#pragma unroll
        for (int k = 0; k < L::NCH; ++k) s[n] = mma(L::row(Q, at, 32 * n, k), kf[k], s[n]);
      }
      feed<NB * L::NCH, 1, 3>();
      const float c = BIAS ? 1.f : a.c;
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        if (BIAS) {
          const int lo = key0 + w * 32 - off - rb - 32 * n - 31;
          add_bias<-1, false>(s[n], a.c, lut, key - off - rb - 32 * n, lo, lo + 62, h, R);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f4 x = *reinterpret_cast<const f4*>(lse + 32 * n + 8 * q + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][4 * q + e] = __builtin_amdgcn_exp2f(fmaf(s[n][4 * q + e], c, -x[e]));
        }
        if (rb + 32 * n < wlast) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (rb + 32 * n + acc_row(r, h) < see) s[n][r] = 0.f;
        }
#pragma unroll
        for (int t = 0; t < L::TB; ++t) {
          const auto pf = take<T>(s[n], t);
#pragma unroll
          for (int dt = 0; dt < L::DT; ++dt) dv[dt] = mma(L::col(G, at, 32 * n, t, dt), pf, dv[dt]);
        }
        feed<L::DT * L::TB, L::CR, 3>();
        __builtin_amdgcn_sched_barrier(0);                     // (merged with the next stage it spills)
#pragma unroll
        for (int q = 0; q < 4; ++q) {                          // dP starts from -delta
          const f4 x = *reinterpret_cast<const f4*>(dl + 32 * n + 8 * q + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) g[n][4 * q + e] = x[e];
        }
#pragma unroll
        for (int k = 0; k < L::NCH; ++k) {
          if constexpr (VL) g[n] = mma(L::row(G, at, 32 * n, k), L::row(vt, at, w * 32, k), g[n]);
          else g[n] = mma(L::row(G, at, 32 * n, k), vf[k], g[n]);
        }
        feed<L::NCH, VL ? 2 : 1, VL ? 2 : 3>();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[n][r] *= g[n][r];
        if (HALF) fit(s[n], power, dk);
#pragma unroll
        for (int t = 0; t < L::TB; ++t) {
          add_ds<L>(dk, Q, at, 32 * n, t, s[n]);
        }
        feed<L::DT * L::TB, L::CR, 3, HALF ? 2 : 1>();
      }
    }
    if (it + 1 < t1) commit(1 - b);
    __syncthreads();
  };
  for (int it = t0; it < t1; it += 2) {
    step(it, Int<0>{});
    if (it + 1 < t1) step(it + 1, Int<1>{});
  }
  if (!valid) return;
  const int64_t rid = (k0 + key) * a.p.Hkv + kvh, rows = a.p.total_k * a.p.Hkv;
  if (nsplit == 1) {
    store_col(reinterpret_cast<T*>(a.p.dk) + rid * D, dk, a.p.scale * power.up * UNLIFT, D, h);
    store_col(reinterpret_cast<T*>(a.p.dv) + rid * D, dv, UNLIFT, D, h);
  } else {
    store_col(a.part_k + ((int64_t)part_no * rows + rid) * D, dk, a.p.scale * power.up * UNLIFT, D, h);
    store_col(a.part_k + ((int64_t)(nsplit + part_no) * rows + rid) * D, dv, UNLIFT, D, h);
  }
}

// -------------------------------------------------------------------------------------------
// backward: both in one launch.  They need nothing of each other but rowsum(dO O), which
// delta_kernel takes first, and share the chip to the end instead of each leaving it half empty (training with 12 heads of 64, up to
// 2047 tokens, dS in one part: dQ 81 and dK / dV 70 us one after the other, 102 together; 10 k tokens, 16 heads of 128 over 4:
// 818 and 765 us, 0.68 TFLOP counted as seven products: 0.89 PFLOP/s)
// -------------------------------------------------------------------------------------------
template <class T, int DP, bool BIAS, int NW>
__global__ __launch_bounds__(NW * 64, (occ_bwd<T, DP, BIAS, NW>())) void bwd_kernel(Args a) {
  const int id = blockIdx.x, nk = a.wgs_k * a.split_k;
  if (id < nk) dkv_body<T, DP, BIAS, NW>(a, id % a.wgs_k, id / a.wgs_k);
  else dq_body<T, DP, BIAS, NW>(a, (id - nk) % a.wgs_q, (id - nk) / a.wgs_q);
}

// delta[row] = sum dO O over the features, 16 lanes a row, 64 tokens of one head a workgroup
template <class T> __global__ __launch_bounds__(256) void delta_kernel(Args a) {
  constexpr int EPC = 16 / sizeof(T);
  const int head = blockIdx.y, l = threadIdx.x & 15, D = a.p.D;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t tok = (int64_t)blockIdx.x * 64 + i * 16 + (threadIdx.x >> 4);
    float x = 0.f;
    if (tok < a.p.total_q) {
      const T* g = reinterpret_cast<const T*>(a.p.dout) + tok * a.p.do_ts + head * a.p.do_hs;
      const T* o = reinterpret_cast<const T*>(a.p.o) + (tok * a.p.Hq + head) * D;
#pragma unroll
      for (int j = 0; j < 128 / (16 * EPC); ++j) {
        const int d = (16 * j + l) * EPC;
        if (d >= D) continue;
        const auto gv = *reinterpret_cast<const typename Ty<T>::Frag*>(g + d);
        const auto ov = *reinterpret_cast<const typename Ty<T>::Frag*>(o + d);
#pragma unroll
        for (int e = 0; e < EPC; ++e) x = fmaf((float)gv[e], (float)ov[e], x);
      }
    }
    x += dpp_mov<0x128>(x);                                    // over the row's 16 lanes
    x += dpp_mov<0x124>(x);
    x += dpp_mov<0x4e>(x);
    x += dpp_mov<0xb1>(x);
    if (tok < a.p.total_q && l == 0) a.delta[tok * a.p.Hq + head] = x;
  }
}

// ---- host: one launcher per type (packed_attention_<type>.hip) ------------------------------
struct Plan {
  Args a;
  int dp, nwq, nwk;            // waves of a workgroup over queries, over keys (backward: the same)
  int64_t hist_bytes;
};
template <class T> int run_fwd(const Plan& p, hipStream_t s);
template <class T> int run_bwd(const Plan& p, hipStream_t s);

template <class T, class K> int launch(K kernel, dim3 grid, int threads, size_t lds, const Args& a, hipStream_t s) {
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL(kernel, grid, dim3(threads), lds, s, a);
  VAESNE_CHECK_LAUNCH();
  return 0;
}

template <class T, int DP, bool BIAS> int fwd_dp(const Plan& p, hipStream_t s) {
  const Args& a = p.a;
  const size_t lds = 4 * (p.nwq == 2 ? key_tile<T, DP, 2>() : key_tile<T, DP, 4>()) * Tile<T, DP>::RB + (BIAS ? span_of(a.p.max_distance) * 4 : 0);
  const int rc = p.nwq == 2 ? launch<T>(fwd_kernel<T, DP, BIAS, 2>, dim3(a.wgs_q, a.split_q), 128, lds, a, s)
                            : launch<T>(fwd_kernel<T, DP, BIAS, 4>, dim3(a.wgs_q, a.split_q), 256, lds, a, s);
  if (rc || a.split_q == 1) return rc;
  const int64_t rows = a.p.total_q * a.p.Hq;
  hipLaunchKernelGGL((join_kernel<T, true>), dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, s, a.part, a.part_lse, a.split_q,
                     rows, a.p.D, reinterpret_cast<T*>(a.p.o), nullptr, a.p.lse);
  VAESNE_CHECK_LAUNCH();
  return 0;
}

// out[i] = part[i] + part[n + i] + ..., in this order
__global__ __launch_bounds__(256) void add_parts_kernel(const float* part, int parts, int64_t n, float* out);

template <class T, int DP> int row_dp(const Plan& p, hipStream_t s) {
  const Args& a = p.a;
  const int nw = p.nwq, split = a.split_r;
  const size_t lds = 4 * (nw == 2 ? key_tile<T, DP, 2>() : key_tile<T, DP, 4>()) * Tile<T, DP>::RB + span_of(a.p.max_distance) * 4;
  float* out = split > 1 ? a.part_delta : a.delta;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(nw == 2 ? reinterpret_cast<const void*>(row_kernel<T, DP, 2>)
                                                     : reinterpret_cast<const void*>(row_kernel<T, DP, 4>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return (int)e;
  }
  if (nw == 2) hipLaunchKernelGGL((row_kernel<T, DP, 2>), dim3(a.wgs_q, split), dim3(128), lds, s, a, out);
  else hipLaunchKernelGGL((row_kernel<T, DP, 4>), dim3(a.wgs_q, split), dim3(256), lds, s, a, out);
  VAESNE_CHECK_LAUNCH();
  if (split > 1) {
    const int64_t n = a.p.total_q * a.p.Hq;
    hipLaunchKernelGGL(add_parts_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a.part_delta, split, n, a.delta);
    VAESNE_CHECK_LAUNCH();
  }
  return 0;
}

template <class T, int DP, bool BIAS> int bwd_dp(const Plan& p, hipStream_t s) {
  const Args& a = p.a;
  constexpr int BQ = row_tile<T, DP>(), RB = Tile<T, DP>::RB;
  const int R = a.p.max_distance, NH = 2 * R + 1, nw = p.nwq, BN = nw == 2 ? key_tile<T, DP, 2>() : key_tile<T, DP, 4>();
  const int64_t blocks = (a.p.total_q + 63) / 64;
  if (BIAS && __is_same(T, __bf16) && a.p.dtable) {
    if (a.wgs_q > 0)
      if constexpr (__is_same(T, __bf16)) {
        const int rc = row_dp<T, DP>(p, s);
        if (rc) return rc;
      }
  } else if (blocks > 0) {
    hipLaunchKernelGGL((delta_kernel<T>), dim3((unsigned)blocks, a.p.Hq), dim3(256), 0, s, a);
    VAESNE_CHECK_LAUNCH();
  }
  const size_t lds_q = 4 * BN * RB + (BIAS ? ((1 + nw) * span_of(R) + 3) / 4 * 16 : 0) + (BIAS && a.p.dtable ? nw * SKEW * 4 : 0);
  const size_t lds_k = 4 * BQ * RB + 16 * BQ + (BIAS ? (span_of(R) * 4 + 15) / 16 * 16 : 0) +
                       (v_in_lds<T, DP>() ? nw * 32 * RB : 0);
  const size_t lds = lds_q > lds_k ? lds_q : lds_k;
  const int wgs = a.wgs_k * a.split_k + a.wgs_q * a.split_q;
  if (wgs > 0) {
    const int rc = nw == 2 ? launch<T>(bwd_kernel<T, DP, BIAS, 2>, dim3(wgs), 128, lds, a, s)
                           : launch<T>(bwd_kernel<T, DP, BIAS, 4>, dim3(wgs), 256, lds, a, s);
    if (rc) return rc;
  }
  if (a.split_q > 1) {
    const int64_t rows = a.p.total_q * a.p.Hq;
    hipLaunchKernelGGL((join_kernel<T, false>), dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, s, a.part, nullptr, a.split_q,
                       rows, a.p.D, reinterpret_cast<T*>(a.p.dq), nullptr, nullptr);
    VAESNE_CHECK_LAUNCH();
  }
  if (a.split_k > 1) {
    const int64_t rows = a.p.total_k * a.p.Hkv;
    hipLaunchKernelGGL((join_kernel<T, false>), dim3((unsigned)((rows + 7) / 8), 2), dim3(256), 0, s, a.part_k, nullptr,
                       a.split_k, rows, a.p.D, reinterpret_cast<T*>(a.p.dk), reinterpret_cast<T*>(a.p.dv), nullptr);
    VAESNE_CHECK_LAUNCH();
  }
  if (BIAS && a.p.dtable) {
    float* rel = a.hist + p.hist_bytes / 4;
    hipLaunchKernelGGL(hist_sum_kernel, dim3((NH + 63) / 64, a.p.Hq), dim3(1024), 0, s, a.hist, a.p.n_q_tiles * a.split_q,
                       a.p.Hq, NH, rel);
    VAESNE_CHECK_LAUNCH();
    hipLaunchKernelGGL((hist_bucket_kernel<T>), dim3(a.p.Hq), dim3(1024), 0, s, rel, a.p.lut, NH, a.p.Hq,
                       a.p.num_buckets, reinterpret_cast<T*>(a.p.dtable));
    VAESNE_CHECK_LAUNCH();
  }
  return 0;
}

template <class T, bool BWD> int dispatch(const Plan& p, hipStream_t s) {
#define VAESNE_PK(DPV)                                                                          \
  if (p.dp == DPV) {                                                                            \
    if constexpr (BWD) return p.a.p.table ? bwd_dp<T, DPV, true>(p, s) : bwd_dp<T, DPV, false>(p, s); \
    else return p.a.p.table ? fwd_dp<T, DPV, true>(p, s) : fwd_dp<T, DPV, false>(p, s);         \
  }
  VAESNE_PK(16) VAESNE_PK(32) VAESNE_PK(64) VAESNE_PK(128)
#undef VAESNE_PK
  return (int)hipErrorInvalidValue;
}

}  // namespace pk
}  // namespace vaesne
