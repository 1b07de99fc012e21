// Root-mean-square norm with the residual's addition and a result in 8 bits (e4m3) with a scale a row:
//   s = a + residual,  rms = sqrt(mean s^2 + eps),  p = s w  (the norm's result is p / rms)
//   D = max(max|p|, 448 * 2^-126 * rms),  q = e4m3(448 p / D),  scale = D / (448 rms)
// and the same without the norm (rms = 1, w = 1) for rows as they are.  rms cancels in q, so q depends on one quotient alone.
//
// A result of 3 mantissa bits meets a tie, or comes near one, in a few values of every million, and 32-bit arithmetic would
// round those by its own errors.  s, p and the quotient are therefore formed in 64 bits: sums and products of two 24-bit
// values are exact there, the quotient gets one Newton step (correctly rounded, exact where it has 53 bits), and it goes to
// 32 bits by rounding to odd, so that the last rounding, to e4m3, is the only one.  One read of each input, one write of
// each result: HBM bounds it.
//
// A row is one wave's (up to 64 pieces of 16 bytes each lane) or four waves'; its inputs stay in registers between the pass
// that sums and the pass that writes.  Longer rows are read again.  A row with a NaN or an infinity in p has the scale NaN
// and q NaN everywhere; its s is what it is.
#include "vmi_dispatch.h"
#include "vmi_vec.h"

using namespace vmi;

namespace {

constexpr int NTH = 256;
constexpr double kTop = 448.0, kLeast = 0x1p-126;

struct Args {
  const void *a, *r, *w;
  int64_t a_stride, r_stride;
  float eps;
  int norm;
  void* sum;
  uint8_t* q;
  float* scale;
  int64_t rows;
  int d;
};

// r (at most 448) to the 32-bit value that any later rounding to fewer bits takes as r itself.
__device__ __forceinline__ float round_to_odd(double r) {
  const float f = static_cast<float>(r);
  const double e = r - static_cast<double>(f);
  uint32_t b = __float_as_uint(f);
  if (e != 0.0 && (b & 1u) == 0u) b += (e > 0.0) == (r > 0.0) ? 1u : ~0u;
  return __uint_as_float(b);
}

template <typename T, typename W> struct Piece {
  static constexpr int N = Vec<T>::N;
  // p and s of the N elements from i0
  static __device__ __forceinline__ void terms(const float (&a)[N], const float (&r)[N], const float (&w)[N], double (&s)[N], double (&p)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      s[j] = static_cast<double>(a[j]) + static_cast<double>(r[j]);
      p[j] = s[j] * static_cast<double>(w[j]);
    }
  }
};

template <typename T, typename W, int N>
__device__ __forceinline__ void load_weights(const W* w, int i0, int d, bool vec, float (&x)[N]) {
  if (w == nullptr) {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = 1.f;
  } else if (vec) {
    typedef typename native<W>::type E;
    typedef E P __attribute__((ext_vector_type(N)));
    const P v = *reinterpret_cast<const P*>(w + i0);
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = static_cast<float>(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = i0 + j < d ? io<W>::load(w, i0 + j) : 0.f;
  }
}

// G threads a row, NV pieces each; LONG: any number of pieces, read again for the second pass.
template <typename T, typename W, int G, int NV, bool LONG, bool VEC>
__global__ __launch_bounds__(NTH) void norm_quant_kernel(Args k) {
  constexpr int N = Vec<T>::N, WAVES = G / 64;
  __shared__ double red[3][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = threadIdx.x % G;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (NTH / G) + threadIdx.x / G;
  if (G < NTH && row >= k.rows) return;
  const T* ar = static_cast<const T*>(k.a) + row * k.a_stride;
  const T* rr = k.r == nullptr ? nullptr : static_cast<const T*>(k.r) + row * k.r_stride;
  const W* w = static_cast<const W*>(k.w);
  T* sr = k.sum == nullptr ? nullptr : static_cast<T*>(k.sum) + row * k.d;
  float a[LONG ? 1 : NV][N], r[LONG ? 1 : NV][N];
  auto load = [&](int i0, float (&x)[N], float (&y)[N]) {
    load_piece<T>(ar, i0, k.d, VEC, x);
    if (rr != nullptr) {
      load_piece<T>(rr, i0, k.d, VEC, y);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) y[j] = 0.f;
    }
  };
  double ss = 0.0, top = 0.0;
  bool bad = false;
  auto gather = [&](int i0, const float (&x)[N], const float (&y)[N]) {
    float wt[N], st[N];
    double s[N], p[N];
    load_weights<T, W, N>(w, i0, k.d, VEC, wt);
    Piece<T, W>::terms(x, y, wt, s, p);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      st[j] = static_cast<float>(s[j]);
      ss += s[j] * s[j];
      top = fmax(top, fabs(p[j]));
      bad |= !(fabs(p[j]) <= 1.7976931348623157e308);
    }
    if (sr != nullptr) store_piece<T>(sr, i0, k.d, VEC, st);
  };
  if constexpr (LONG) {
    for (int i0 = g * N; i0 < k.d; i0 += G * N) {
      load(i0, a[0], r[0]);
      gather(i0, a[0], r[0]);
    }
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (const int i0 = (v * G + g) * N; i0 < k.d) load(i0, a[v], r[v]);
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (const int i0 = (v * G + g) * N; i0 < k.d) gather(i0, a[v], r[v]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    ss += __shfl_xor(ss, o);
    top = fmax(top, __shfl_xor(top, o));
  }
  bad = __any(bad);
  if constexpr (WAVES > 1) {
    if (lane == 0) red[0][wave] = ss, red[1][wave] = top, red[2][wave] = bad ? 1.0 : 0.0;
    __syncthreads();
    ss = red[0][0] + red[0][1] + red[0][2] + red[0][3];
    top = fmax(fmax(red[1][0], red[1][1]), fmax(red[1][2], red[1][3]));
    bad = red[2][0] + red[2][1] + red[2][2] + red[2][3] != 0.0;
  }
  const double rms = k.norm ? sqrt(ss / k.d + static_cast<double>(k.eps)) : 1.0;
  const double D = fmax(top, kTop * kLeast * rms), inv = 1.0 / D;
  if (g == 0) k.scale[row] = bad ? __builtin_nanf("") : static_cast<float>(D / (kTop * rms));
  uint8_t* qr = k.q + row * k.d;
  auto write = [&](int i0, const float (&x)[N], const float (&y)[N]) {
    float wt[N], f[N];
    double s[N], p[N];
    load_weights<T, W, N>(w, i0, k.d, VEC, wt);
    Piece<T, W>::terms(x, y, wt, s, p);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const double t = kTop * p[j], q0 = t * inv;
      f[j] = round_to_odd(fma(fma(-q0, D, t), inv, q0));
      if (bad) f[j] = __builtin_nanf("");
    }
    uint32_t packed[N / 4];
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      int u = __builtin_amdgcn_cvt_pk_fp8_f32(f[j], f[j + 1], 0, false);
      packed[j / 4] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(f[j + 2], f[j + 3], u, true));
    }
    if (VEC) {
#pragma unroll
      for (int j = 0; j < N / 4; ++j) reinterpret_cast<uint32_t*>(qr + i0)[j] = packed[j];
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (i0 + j < k.d) qr[i0 + j] = static_cast<uint8_t>(packed[j / 4] >> (8 * (j % 4)));
    }
  };
  if constexpr (LONG) {
    for (int i0 = g * N; i0 < k.d; i0 += G * N) {
      load(i0, a[0], r[0]);
      write(i0, a[0], r[0]);
    }
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (const int i0 = (v * G + g) * N; i0 < k.d) write(i0, a[v], r[v]);
  }
}

template <typename T, typename W, int G, int NV, bool LONG> int launch(Args k, bool vec, hipStream_t stream) {
  return in_launches(k.rows, NTH, NTH / G, [&](int64_t row, int64_t n) -> int {
    Args c = k;
    c.a = advance<const T>(k.a, row * k.a_stride), c.r = advance<const T>(k.r, row * k.r_stride);
    c.sum = advance<T>(k.sum, row * k.d), c.q = k.q + row * k.d, c.scale = k.scale + row, c.rows = n;
    const dim3 grid(static_cast<unsigned>((n + NTH / G - 1) / (NTH / G)));
    if (vec)
      hipLaunchKernelGGL((norm_quant_kernel<T, W, G, NV, LONG, true>), grid, dim3(NTH), 0, stream, c);
    else
      hipLaunchKernelGGL((norm_quant_kernel<T, W, G, NV, LONG, false>), grid, dim3(NTH), 0, stream, c);
    return hip_status(hipGetLastError());
  });
}

template <typename T, typename W> int by_row(const Args& k, bool vec, hipStream_t stream) {
  const int pieces = (k.d + Vec<T>::N - 1) / Vec<T>::N;
  if (pieces <= 64) return launch<T, W, 64, 1, false>(k, vec, stream);
  if (pieces <= 128) return launch<T, W, 64, 2, false>(k, vec, stream);
  if (pieces <= 256) return launch<T, W, 64, 4, false>(k, vec, stream);
  if (pieces <= 512) return launch<T, W, 64, 8, false>(k, vec, stream);
  if (pieces <= 1024) return launch<T, W, 256, 4, false>(k, vec, stream);
  if (pieces <= 2048) return launch<T, W, 256, 8, false>(k, vec, stream);
  return launch<T, W, 256, 1, true>(k, vec, stream);
}

}  // namespace

extern "C" int vmi_norm_add_quant(const void* a, int64_t a_stride, const void* residual, int64_t r_stride, const void* w, int dtype,
                                  int w_dtype, int norm, float eps, void* sum, void* q, float* scale, int64_t rows, int64_t d,
                                  void* stream) {
  if (rows < 0 || d < 1 || d > INT32_MAX - 65536 || dtype < 0 || dtype > VMI_F16 || (w_dtype != dtype && w_dtype != VMI_F32))
    return VMI_ERR_INVALID_ARG;
  if (rows == 0) return VMI_OK;
  if (a == nullptr || q == nullptr || scale == nullptr) return VMI_ERR_INVALID_ARG;
  Args k{a, residual, w, a_stride, residual == nullptr ? 0 : r_stride, eps, norm, sum, static_cast<uint8_t*>(q), scale, rows,
         static_cast<int>(d)};
  return by_type(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    const bool vec = d % Vec<T>::N == 0 && k.a_stride % Vec<T>::N == 0 && k.r_stride % Vec<T>::N == 0 && aligned16({a, residual, w, sum}) &&
                     reinterpret_cast<uintptr_t>(q) % 4 == 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if constexpr (sizeof(T) == 2)
      if (w != nullptr && w_dtype == VMI_F32) return by_row<T, float>(k, vec, s);
    return by_row<T, T>(k, vec, s);
  });
}
