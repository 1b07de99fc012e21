// Root-mean-square norm with the residual's addition and a result in 8 bits (e4m3) with a scale a row:
//   s = a + residual,  rms = sqrt(mean s^2 + eps),  p = s w  (the norm's result is p / rms)
//   D = max(max|p|, 448 * 2^-126 * rms),  q = e4m3(448 p / D),  scale = D / (448 rms)
// and the same without the norm (rms = 1, w = 1) for rows as they are.  rms cancels in q, so q depends on one quotient alone.
//
// A result of 3 mantissa bits meets a tie, or comes near one, in a few values of every million, and 32-bit arithmetic would
// round those by its own errors.  In 64 bits s and p are exact (sums and products of two 24-bit values), and the quotient with
// one Newton step is correctly rounded, exact where it has 53 bits; it goes to 32 bits by rounding to odd, so that the rounding
// to e4m3 is the only one.  That is needed where the 32-bit quotient, four roundings of 2^-24 off, lies within 16 of its steps
// of a tie (and below 2^-6, where e4m3's steps are of one size): one value of about 5000, so a wave takes the 64-bit form for
// a whole piece where one of its lanes needs it.  max|p| in 64 bits is that of the pieces whose 32-bit maximum is within
// 2^-21 of the row's.  Rows whose 32-bit terms are not all finite, or all below 2^-60, take the 64-bit form throughout.
// The sum of squares is of 64 bits, over s of 32 for 16-bit inputs (of 64 in the rows above): the scale is within 2^-23.
//
// One read of each input, one write of each result: HBM bounds it.  A row is one wave's (up to 4 pieces of 16 bytes a lane)
// or four waves'; its inputs stay in registers, as they came, between the pass that sums and the pass that writes.  Longer rows
// are read again.  A row with a NaN or an infinity in p has the scale NaN and q NaN everywhere; its s is what it is.
#include <type_traits>

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

// Pieces of a row start where the row does; the hardware takes 16 bytes at any address.
template <typename W, int N, bool WHOLE> __device__ __forceinline__ void load_weights(const W* w, int i0, int d, float (&x)[N]) {
  if (w == nullptr) {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = 1.f;
  } else if (WHOLE || i0 + N <= d) {
    W v[N];
    __builtin_memcpy(v, w + i0, sizeof(v));
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = io<W>::to_f32(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = i0 + j < d ? io<W>::load(w, i0 + j) : 0.f;
  }
}

// 16 bytes of a row from element i0 as they lie, zeros past its end.  ONCE: nothing reads them again (32768 x 4096 bf16 with
// these loads 189 us, with ordinary ones 241: the results then keep more of the caches).
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(1)));
template <typename T, bool WHOLE, bool ONCE> __device__ __forceinline__ Vec<T> load_raw(const T* row, int i0, int d) {
  Vec<T> v;
  if (WHOLE || i0 + Vec<T>::N <= d) {
    const u32x4_any* from = reinterpret_cast<const u32x4_any*>(row + i0);
    const u32x4 x = ONCE ? __builtin_nontemporal_load(from) : *from;
    return __builtin_bit_cast(Vec<T>, x);
  }
#pragma unroll
  for (int j = 0; j < Vec<T>::N; ++j) {
    if (i0 + j < d) v.e[j] = row[i0 + j];
    else io<T>::store(v.e, j, 0.f);
  }
  return v;
}
template <typename T, bool WHOLE> __device__ __forceinline__ void store_sum(T* row, int i0, int d, const float (&x)[Vec<T>::N]) {
  typename native<T>::type e[Vec<T>::N];
#pragma unroll
  for (int j = 0; j < Vec<T>::N; ++j) e[j] = static_cast<typename native<T>::type>(x[j]);
  if (WHOLE || i0 + Vec<T>::N <= d) {
    __builtin_memcpy(row + i0, e, 16);
  } else {
#pragma unroll
    for (int j = 0; j < Vec<T>::N; ++j)
      if (i0 + j < d) __builtin_memcpy(row + i0 + j, e + j, sizeof(T));
  }
}

// The terms of one piece in 32 bits and, where it matters, in 64.  Sums of two 16-bit values are exact in 32 bits, but where
// one is 2^16 times the other and more.
template <typename T, bool RES> struct Terms {
  static constexpr int N = Vec<T>::N;
  Vec<T> a, r;
  float w[N];
  __device__ __forceinline__ float s(int j) const {
    const float x = io<T>::to_f32(a.e[j]);
    return RES ? x + io<T>::to_f32(r.e[j]) : x;
  }
  __device__ __forceinline__ double s64(int j) const {
    const double x = io<T>::to_f32(a.e[j]);
    return RES ? x + static_cast<double>(io<T>::to_f32(r.e[j])) : x;
  }
  __device__ __forceinline__ float p(int j) const { return s(j) * w[j]; }
  __device__ __forceinline__ double p64(int j) const { return s64(j) * static_cast<double>(w[j]); }
};

// Keeps the compiler from carrying a piece's terms from one pass to the next in registers (8 a piece of 16 bits):
// they are formed again from the 16 bytes.
template <typename T> __device__ __forceinline__ void forget(Vec<T>& v) {
  u32x4 x = __builtin_bit_cast(u32x4, v);
  asm volatile("" : "+v"(x));
  v = __builtin_bit_cast(Vec<T>, x);
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}

// G threads a row, NV pieces each; LONG: any number of pieces, read again for the second pass; RES: with a residual; WHOLE: rows
// are whole pieces (a row's last piece otherwise goes element by element).
template <typename T, typename W, int G, int NV, bool LONG, bool RES, bool WHOLE>
__global__ __launch_bounds__(NTH) void norm_quant_kernel(Args k) {
  constexpr int N = Vec<T>::N, WAVES = G / 64;
  __shared__ double red[2][4];
  __shared__ float red32[2][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = threadIdx.x % G;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (NTH / G) + threadIdx.x / G;
  if (G < NTH && row >= k.rows) return;
  const T* ar = static_cast<const T*>(k.a) + row * k.a_stride;
  const T* rr = static_cast<const T*>(k.r) + (RES ? row * k.r_stride : 0);
  const W* w = static_cast<const W*>(k.w);
  T* sr = k.sum == nullptr ? nullptr : static_cast<T*>(k.sum) + row * k.d;
  Vec<T> a[LONG ? 1 : NV] = {}, r[LONG ? 1 : NV] = {};
  auto load = [&](int v, int i0) {
    a[v] = load_raw<T, WHOLE, !LONG>(ar, i0, k.d);
    if constexpr (RES) r[v] = load_raw<T, WHOLE, !LONG>(rr, i0, k.d);
  };
  auto terms = [&](int v, int i0) {
    Terms<T, RES> t;
    t.a = a[v], t.r = r[v];
    load_weights<W, N, WHOLE>(w, i0, k.d, t.w);
    return t;
  };
  // f(v, i0) for each of the thread's pieces, `again`: after another pass over them
  auto pieces = [&](bool again, auto&& f) {
    if constexpr (LONG) {
      for (int i0 = g * N; i0 < k.d; i0 += G * N) {
        load(0, i0);
        f(0, i0);
      }
    } else {
      if (!again) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
          if (const int i0 = (v * G + g) * N; i0 < k.d) load(v, i0);
      } else {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          forget(a[v]);
          if constexpr (RES) forget(r[v]);
        }
      }
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (const int i0 = (v * G + g) * N; i0 < k.d) f(v, i0);
    }
  };
  double ss = 0.0;
  float odd = 0.f, high = 0.f, of_piece[LONG ? 1 : NV];  // odd: NaN after a NaN or an infinity
#pragma unroll
  for (int v = 0; v < (LONG ? 1 : NV); ++v) of_piece[v] = 0.f;
  pieces(false, [&](int v, int i0) {
    const Terms<T, RES> t = terms(v, i0);
    float st[N], m = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const double s = sizeof(T) == 2 ? static_cast<double>(t.s(j)) : t.s64(j);
      const float p = t.p(j);
      st[j] = static_cast<float>(s);
      ss += s * s;
      m = fmaxf(m, fabsf(p));
      odd = fmaf(p, 0.f, odd);
    }
    high = fmaxf(high, m);
    of_piece[v] = m;
    if (sr != nullptr) store_sum<T, WHOLE>(sr, i0, k.d, st);
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
  high = wave_max(high);
  bool wild = __any(!(odd == 0.f));
  if constexpr (WAVES > 1) {
    if (lane == 0) red[0][wave] = ss, red32[0][wave] = high, red32[1][wave] = wild ? 1.f : 0.f;
    __syncthreads();
    ss = red[0][0] + red[0][1] + red[0][2] + red[0][3];
    high = fmaxf(fmaxf(red32[0][0], red32[0][1]), fmaxf(red32[0][2], red32[0][3]));
    wild = red32[1][0] + red32[1][1] + red32[1][2] + red32[1][3] != 0.f;
  }
  wild = wild || high < 0x1p-60f;
  // the largest |p| in 64 bits
  const float near = wild ? -1.f : high * (1.f - 0x1p-21f);
  double top = 0.0, again = 0.0;
  bool bad = false;
  // a bf16 row's sums may lie beyond fp32: their squares are then summed again, in 64 bits throughout
  constexpr bool AGAIN = RES && std::is_same<T, bf16_t>::value;
  pieces(true, [&](int v, int i0) {
    if (LONG || __any(of_piece[v] >= near)) {
      const Terms<T, RES> t = terms(v, i0);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const double p = fabs(t.p64(j));
        top = fmax(top, p);
        bad |= !(p <= 1.7976931348623157e308);
      }
      if (AGAIN && wild) {
#pragma unroll
        for (int j = 0; j < N; ++j) again += t.s64(j) * t.s64(j);
      }
    }
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmax(top, __shfl_xor(top, o));
  bad = __any(bad);
  if (AGAIN && wild) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) again += __shfl_xor(again, o);
    ss = again;
  }
  if constexpr (WAVES > 1) {
    __syncthreads();
    if (lane == 0) red[0][wave] = again, red[1][wave] = top, red32[0][wave] = bad ? 1.f : 0.f;
    __syncthreads();
    if (AGAIN && wild) ss = red[0][0] + red[0][1] + red[0][2] + red[0][3];
    top = fmax(fmax(red[1][0], red[1][1]), fmax(red[1][2], red[1][3]));
    bad = red32[0][0] + red32[0][1] + red32[0][2] + red32[0][3] != 0.f;
  }
  const double rms = k.norm ? sqrt(ss / k.d + static_cast<double>(k.eps)) : 1.0;
  const double D = fmax(top, kTop * kLeast * rms), inv = 1.0 / D;
  const float F = static_cast<float>(kTop * inv);
  if (g == 0) k.scale[row] = bad ? __builtin_nanf("") : static_cast<float>(D / (kTop * rms));
  uint8_t* qr = k.q + row * k.d;
  pieces(true, [&](int v, int i0) {
    const Terms<T, RES> t = terms(v, i0);
    float f[N];
    // how far above 16 steps before the middle between two values (the low 20 bits half way), and above the least 32-bit value
    uint32_t middle = ~0u, least = ~0u;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      f[j] = t.p(j) * F;
      const uint32_t u = __float_as_uint(f[j]);
      middle = min(middle, (u << 12) - 0x7FFF0000u);
      least = min(least, (u << 1) - 2u);
    }
    const bool doubt = wild || middle <= 0x20000u || least < 0x79000000u - 2u;  // 0x3C800000 is 2^-6
    if (__any(doubt)) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const double x = kTop * t.p64(j), q0 = x * inv;
        f[j] = bad ? __builtin_nanf("") : round_to_odd(fma(fma(-q0, D, x), inv, q0));
      }
    }
    uint32_t packed[N / 4];
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      int u = __builtin_amdgcn_cvt_pk_fp8_f32(f[j], f[j + 1], 0, false);
      packed[j / 4] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(f[j + 2], f[j + 3], u, true));
    }
    if (WHOLE || i0 + N <= k.d) {
      __builtin_memcpy(qr + i0, packed, N);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (i0 + j < k.d) qr[i0 + j] = static_cast<uint8_t>(packed[j / 4] >> (8 * (j % 4)));
    }
  });
}

template <typename T, typename W, int G, int NV, bool LONG> int launch(const Args& k, hipStream_t stream) {
  return in_launches(k.rows, NTH, NTH / G, [&](int64_t row, int64_t n) -> int {
    Args c = k;
    c.a = advance<const T>(k.a, row * k.a_stride), c.r = advance<const T>(k.r, row * k.r_stride);
    c.sum = advance<T>(k.sum, row * k.d), c.q = k.q + row * k.d, c.scale = k.scale + row, c.rows = n;
    const dim3 grid(static_cast<unsigned>((n + NTH / G - 1) / (NTH / G)));
    auto go = [&](auto res, auto whole) {
      hipLaunchKernelGGL((norm_quant_kernel<T, W, G, NV, LONG, decltype(res)::value, decltype(whole)::value>), grid, dim3(NTH), 0,
                         stream, c);
    };
    const std::true_type yes;
    const std::false_type no;
    const bool whole = k.d % Vec<T>::N == 0;
    if (k.r != nullptr) whole ? go(yes, yes) : go(yes, no);
    else whole ? go(no, yes) : go(no, no);
    return hip_status(hipGetLastError());
  });
}

template <typename T, typename W> int by_row(const Args& k, hipStream_t stream) {
  const int pieces = (k.d + Vec<T>::N - 1) / Vec<T>::N;
  if (pieces <= 64) return launch<T, W, 64, 1, false>(k, stream);
  if (pieces <= 128) return launch<T, W, 64, 2, false>(k, stream);
  if (pieces <= 256) return launch<T, W, 64, 4, false>(k, stream);
  if (pieces <= 512) return launch<T, W, 256, 2, false>(k, stream);  // 189 us for 193 by one wave a row of 8 pieces a lane
  if (pieces <= 1024) return launch<T, W, 256, 4, false>(k, stream);
  if (pieces <= 2048) return launch<T, W, 256, 8, false>(k, stream);
  return launch<T, W, 256, 1, true>(k, stream);
}

}  // namespace

extern "C" int vmi_norm_add_quant(const void* a, int64_t a_stride, const void* residual, int64_t r_stride, const void* w, int dtype,
                                  int w_dtype, int norm, float eps, void* sum, void* q, float* scale, int64_t rows, int64_t d,
                                  void* stream) {
  if (rows < 0 || d < 1 || d > INT32_MAX - 65536 || dtype < 0 || dtype > VMI_F16 || (w_dtype != dtype && w_dtype != VMI_F32))
    return VMI_ERR_INVALID_ARG;
  if (norm && !(eps >= 0.f && eps <= 3.40282347e38f)) return VMI_ERR_INVALID_ARG;
  if (rows == 0) return VMI_OK;
  if (a == nullptr || q == nullptr || scale == nullptr) return VMI_ERR_INVALID_ARG;
  Args k{a, residual, w, a_stride, residual == nullptr ? 0 : r_stride, eps, norm, sum, static_cast<uint8_t*>(q), scale, rows,
         static_cast<int>(d)};
  return by_type(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if constexpr (sizeof(T) == 2)
      if (w != nullptr && w_dtype == VMI_F32) return by_row<T, float>(k, s);
    return by_row<T, T>(k, s);
  });
}
