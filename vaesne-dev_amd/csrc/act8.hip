// Activations kept in 8 bits for the backward pass (include/vaesne_hip.h: vaesne_pack8,
// vaesne_gelu8_*).  A thread holds 8 consecutive values, 4 neighbouring lanes a block of 32; the
// block's largest |x| is an integer maximum of bit patterns over the quad (two DPP moves), which also
// finds infinities and NaN.  The step is a power of two, so scaling, rounding and reading back are
// exact but for the one rounding to a whole code.  Bound by HBM: forward reads x and writes y, the
// codes and 1/32 byte of exponents for each value (8192 x 16384 bf16: 675 MB either way, forward 0.118 ms,
// backward 0.134 ms, 5.7 and 5.0 TB/s; a copy of 1 GiB reaches 5.2).  16 values per thread: backward 0.173 ms instead of
// 0.143; one ldexp per value in place of a product with the block's step: 0.160.
#include "common.h"

using namespace vaesne;

namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef float f8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

template <class T> struct V8;
template <> struct V8<float> { using Vec = f8; };
template <> struct V8<__bf16> { using Vec = b8; };
template <> struct V8<_Float16> { using Vec = h8; };

constexpr int NT = 256;

// 8 values from element i on (VEC: 16-byte aligned tensors; the last values one by one)
template <class T, bool VEC> __device__ __forceinline__ f8 load8(const T* p, int64_t i, int64_t n) {
  if (VEC && i + 8 <= n) {
    typename V8<T>::Vec v;
    u4* r = reinterpret_cast<u4*>(&v);
#pragma unroll
    for (unsigned k = 0; k < sizeof(v) / 16; ++k) r[k] = reinterpret_cast<const u4*>(p + i)[k];
    return __builtin_convertvector(v, f8);
  }
  f8 v;
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = i + k < n ? (float)p[i + k] : 0.f;
  return v;
}
template <class T, bool VEC> __device__ __forceinline__ void store8(T* p, int64_t i, int64_t n, f8 x) {
  if (VEC && i + 8 <= n) {
    const auto v = __builtin_convertvector(x, typename V8<T>::Vec);
    const u4* r = reinterpret_cast<const u4*>(&v);
#pragma unroll
    for (unsigned k = 0; k < sizeof(v) / 16; ++k) reinterpret_cast<u4*>(p + i)[k] = r[k];
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (i + k < n) p[i + k] = (T)x[k];
}

template <int CTRL> __device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
  return o > v ? o : v;
}

__device__ __forceinline__ void encode(f8 x, int64_t i, int64_t n, int8_t* codes, uint8_t* exps) {
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t b = __float_as_uint(x[k]) & 0x7fffffffu;
    top = b > top ? b : top;
  }
  top = quad_max<0xb1>(top);               // lanes l ^ 1, then l ^ 2: the 4 lanes of a block
  top = quad_max<0x4e>(top);
  const int field = (int)(top >> 23), e = field < 1 ? 1 : field;
  u2 w = {0, 0};
  if (e < 255) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int c = (int)fminf(fmaxf(rintf(ldexpf(x[k], 133 - e)), -127.f), 127.f);
      w[k >> 2] |= (uint32_t)(c & 255) << (8 * (k & 3));
    }
  }
  if (i + 8 <= n) {
    *reinterpret_cast<u2*>(codes + i) = w;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) codes[i + k] = (int8_t)(w[k >> 2] >> (8 * (k & 3)));
  }
  if ((i & 31) == 0 && i < n) exps[i >> 5] = (uint8_t)e;
}

__device__ __forceinline__ f8 decode(const int8_t* codes, const uint8_t* exps, int64_t i, int64_t n) {
  f8 v;
  if (i >= n) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.f;
    return v;
  }
  const int e = exps[i >> 5];
  u2 w = {0, 0};
  if (i + 8 <= n) {
    w = *reinterpret_cast<const u2*>(codes + i);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) w[k >> 2] |= (uint32_t)(uint8_t)codes[i + k] << (8 * (k & 3));
  }
  const float step = e == 255 ? __builtin_nanf("") : ldexpf(1.f, e - 133);   // (2^-132 and up: subnormal, exact)
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = (float)(int8_t)(w[k >> 2] >> (8 * (k & 3))) * step;
  return v;
}

// The distribution function erfc(-x / sqrt 2) / 2 and the density's exponential exp(-x^2 / 2), both with their error
// relative to themselves: GELU(x) and its slope shrink with them for negative x (an absolute bound, as published
// formulas have, leaves a bf16 result 9 steps off at -6, and 1 + erf has no digits left there).  The tail below -|x| is
// exp(-x^2 / 2) R(|x|); R, which falls like 1 / |x|, is t times a polynomial in t = 1 / (1 + b |x|) of least
// relative error up to |x| = 14.5.  16-bit results: b = 0.46, degree 5, 8.6e-6 (2^-6 of fp16's half step; forward and
// backward of 8192 x 16384 in bf16 234 us, with degree 4, 3.5e-5, 231.5).  fp32 results: b = 0.8, degree 7 from |x| = 0.95 on, 8e-8, 6 of 2^-24 with its roundings; 1/2 + x times a polynomial in x^2 up to 1; the exponential
// of x^2 in two parts.  Below 2^-126 both are 0.  (fp32 at 8192 x 8192, forward and backward: the library's erff, which loses the
// tail, 103 and 112 us; its erfcf 152 and 173; so 104 and 115.)
template <class T> __device__ __forceinline__ float normal_cdf(float x, float& ex) {
  if constexpr (sizeof(T) == 4) {
    const float u = fminf(fabsf(x), 16.f);           // (further out nothing changes)
    const float h = u * u, a = -0.72134752f * h;     // log2(e) / 2 = 0.72134752 + 9.6e-9
    const float rest = fmaf(-0.72134752f, fmaf(u, u, -h), fmaf(-9.62981517e-09f, h, fmaf(-0.72134752f, h, -a)));
    ex = __builtin_amdgcn_exp2f(a);
    ex = fmaf(ex * rest, 0.69314718f, ex);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.8f, u, 1.f));
    const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.97262383f, -2.8332903f), 3.1880875f), -1.4138918f),
                                                          -0.13490756f), 0.098524183f), 0.32006449f), 0.31913286f);
    const float tail = p * ex;
    const float mid = fmaf(x, fmaf(h, fmaf(h, fmaf(h, fmaf(h, 9.4384544e-05f, -0.0011696537f), 0.0099673858f), -0.066489622f), 0.39894226f), 0.5f);
    return u < 1.f ? mid : x < 0.f ? tail : 1.f - tail;
  } else {
    ex = __builtin_amdgcn_exp2f(-0.5f * 1.4426950408889634f * x * x);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.46f, fabsf(x), 1.f));
    const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.07222806f, -0.23654465f), 0.17780116f), 0.11610668f), 0.1870667f),
                             0.18334633f);
    const float tail = p * ex;
    return x < 0.f ? tail : 1.f - tail;
  }
}
template <class T> __device__ __forceinline__ float gelu8(float x) {
  float ex;
  const float c = normal_cdf<T>(x, ex);
  return x < -14.f ? -0.f : x * c;                   // (-inf: 0, not inf * 0)
}
template <class T> __device__ __forceinline__ float gelu8_grad(float x) {
  float ex;
  const float c = normal_cdf<T>(x, ex);
  return fmaf(x * 0.39894228040143268f, ex, c);
}

template <class T, bool VEC, bool GELU>
__global__ __launch_bounds__(NT) void keep_kernel(const T* __restrict__ x, int64_t n, T* __restrict__ y,
                                                  int8_t* __restrict__ codes, uint8_t* __restrict__ exps) {
  const int64_t i = ((int64_t)blockIdx.x * NT + threadIdx.x) * 8;
  f8 v = load8<T, VEC>(x, i, n);
  if (!GELU || codes) encode(v, i, n, codes, exps);
  if (GELU) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = gelu8<T>(v[k]);
    store8<T, VEC>(y, i, n, v);
  }
}

// GELU: dx (and y_again); else the values themselves into dx
template <class T, bool VEC, bool GELU>
__global__ __launch_bounds__(NT) void back_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ exps,
                                                  const T* __restrict__ dy, int64_t n, T* __restrict__ dx,
                                                  T* __restrict__ y_again) {
  const int64_t i = ((int64_t)blockIdx.x * NT + threadIdx.x) * 8;
  if (i >= n) return;
  f8 v = decode(codes, exps, i, n);
  if (GELU) {
    f8 g = load8<T, VEC>(dy, i, n);
    if (y_again) {
      f8 y;
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = gelu8<T>(v[k]);
      store8<T, VEC>(y_again, i, n, y);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = g[k] * gelu8_grad<T>(v[k]);
  }
  store8<T, VEC>(dx, i, n, v);
}

bool ok16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
dim3 grid_of(int64_t n) { return dim3((unsigned)((n + NT * 8 - 1) / (NT * 8))); }

template <class T, bool GELU> int keep(const void* x, int64_t n, void* y, int8_t* codes, uint8_t* exps, hipStream_t s) {
  const T* xp = reinterpret_cast<const T*>(x);
  T* yp = reinterpret_cast<T*>(y);
  if (ok16(x) && ok16(y)) hipLaunchKernelGGL((keep_kernel<T, true, GELU>), grid_of(n), dim3(NT), 0, s, xp, n, yp, codes, exps);
  else hipLaunchKernelGGL((keep_kernel<T, false, GELU>), grid_of(n), dim3(NT), 0, s, xp, n, yp, codes, exps);
  VAESNE_CHECK_LAUNCH();
  return 0;
}
template <class T, bool GELU>
int back(const int8_t* codes, const uint8_t* exps, const void* dy, int64_t n, void* dx, void* y, hipStream_t s) {
  const T* gp = reinterpret_cast<const T*>(dy);
  T *xp = reinterpret_cast<T*>(dx), *yp = reinterpret_cast<T*>(y);
  if (ok16(dy) && ok16(dx) && ok16(y)) hipLaunchKernelGGL((back_kernel<T, true, GELU>), grid_of(n), dim3(NT), 0, s, codes, exps, gp, n, xp, yp);
  else hipLaunchKernelGGL((back_kernel<T, false, GELU>), grid_of(n), dim3(NT), 0, s, codes, exps, gp, n, xp, yp);
  VAESNE_CHECK_LAUNCH();
  return 0;
}
// codes are stored 8 at a time; an axis of a grid has fewer than 2^32 threads
bool bad(int type, int64_t n, const void* codes) {
  return type < 0 || type > 2 || n < 0 || (reinterpret_cast<uintptr_t>(codes) & 7) || n / (NT * 8) >= (1ll << 24) - 1;
}

template <bool GELU> int keep_any(int type, const void* x, int64_t n, void* y, int8_t* codes, uint8_t* exps, void* stream) {
  if (bad(type, n, codes) || (n > 0 && (!x || (GELU ? !codes != !exps || !y : !codes || !exps)))) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  hipStream_t s = (hipStream_t)stream;
  return type == 0 ? keep<float, GELU>(x, n, y, codes, exps, s)
         : type == 1 ? keep<__bf16, GELU>(x, n, y, codes, exps, s) : keep<_Float16, GELU>(x, n, y, codes, exps, s);
}
template <bool GELU>
int back_any(int type, const int8_t* codes, const uint8_t* exps, const void* dy, int64_t n, void* dx, void* y, void* stream) {
  if (bad(type, n, codes) || (n > 0 && (!dx || !codes || !exps || (GELU && !dy)))) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  hipStream_t s = (hipStream_t)stream;
  return type == 0 ? back<float, GELU>(codes, exps, dy, n, dx, y, s)
         : type == 1 ? back<__bf16, GELU>(codes, exps, dy, n, dx, y, s) : back<_Float16, GELU>(codes, exps, dy, n, dx, y, s);
}

}  // namespace

VAESNE_API int vaesne_pack8(int type, const void* x, int64_t n, int8_t* codes, uint8_t* exps, void* stream) {
  return keep_any<false>(type, x, n, nullptr, codes, exps, stream);
}
VAESNE_API int vaesne_unpack8(int type, const int8_t* codes, const uint8_t* exps, int64_t n, void* x, void* stream) {
  return back_any<false>(type, codes, exps, nullptr, n, x, nullptr, stream);
}
VAESNE_API int vaesne_gelu8_fwd(int type, const void* x, int64_t n, void* y, int8_t* codes, uint8_t* exps, void* stream) {
  return keep_any<true>(type, x, n, y, codes, exps, stream);
}
VAESNE_API int vaesne_gelu8_bwd(int type, const int8_t* codes, const uint8_t* exps, const void* dy, int64_t n, void* dx,
                                void* y_again, void* stream) {
  return back_any<true>(type, codes, exps, dy, n, dx, y_again, stream);
}
