// The feed-forward operators' kernels on the product tiles of product_tile.h: what their epilogues compute, and how their
// launches are chosen.  One file per element type instantiates them (feed_forward_*.hip); feed_forward.hip has the C entries.
#pragma once

#include <type_traits>

#include "product_tile.h"
#include "vmi_dispatch.h"
#include "vmi_vec.h"

namespace vmi {
namespace prod {

enum Kind {
  LINEAR,     // y = residual + act(x W^T + b)
  GATED,      // h = act(x Wg^T) lin(x Wu^T)
  LINEAR_DZ,  // dz = dy act'(x W^T + b)
  GATED_DZ,   // dg = dh act'(g) lin(u), du = dh act(g) lin'(u), side by side
  DX,         // dz W (and for the gated form dg Wg + du Wu)
  DW          // dz^T x, or a share of its rows' sum
};
enum Act { ACT_NONE = 0, ACT_SILU = 1, ACT_GELU = 2, ACT_SITU = 3 };

struct Gate {
  int act;
  float b1, b2, i1, i2;  // i: the inverses
};

struct Args {
  const void* a;     // x, dz
  const void* b;     // the weight, x
  const void* b2;    // the second weight
  int64_t lda, ldb;  // elements
  int m, n, k;       // of the result and the contraction
  int tiles_m, tiles_n, group;
  int splits, split_k;     // DW: shares of the contraction, and their length
  // epilogue
  const float *xs, *ws, *ws2;
  const void* bias;
  const void* other;       // residual, dy, dh
  int64_t ldother;
  void* out;
  int64_t ldo;
  int64_t second;          // GATED_DZ: the first column of du; DX: where the second segment starts in a row of a
  int out_dtype;           // e4m3 operands: the result's
  float* partial;          // DW with several shares
  float* keep;             // LINEAR, GATED: the sums before the activation, [m, n] (GATED [m, 2 n], a row's gates first), or null
  int seg, seg_valid;      // DW: rows of the result come in segments of seg, of which seg_valid are stored
  int act;
  Gate gate;               // the gated kinds
};

template <typename E> struct memory { typedef E type; };
template <> struct memory<__bf16> { typedef bf16_t type; };

// Phi(z), the normal distribution's, and e = exp(-z^2 / 2):
//   Phi(-|z|) = e erfcx(|z| / sqrt 2) / 2,  Phi(|z|) = 1 - Phi(-|z|)
// so that the left tail keeps its own precision (1 + erf is 0 below -5.5).  32-bit results: the library's erfcx, and the exponent in two
// parts, whose second, the rounding of z^2, is a factor.  16-bit results: erfcx(z / sqrt 2) / 2 = t P(t), t = 1 / (1 + 0.325 z), P of
// degree 7 with the least relative error over all z >= 0 (9e-7 in fp32).
struct Normal {
  float cdf, e;
};
template <typename T> __device__ __forceinline__ Normal normal(float z) {
  const float x = fabsf(z), sq = z * z;
  Normal r;
  float tail;
  if constexpr (sizeof(T) == 4) {
    const float low = fmaf(z, z, -sq), e = expf(-0.5f * sq);
    r.e = e > 0.f ? fmaf(-0.5f * low, e, e) : 0.f;  // far out z^2 is infinite, and low no number
    tail = 0.5f * erfcxf(x * 0.707106781f) * r.e;
  } else {
    r.e = __builtin_amdgcn_exp2f(sq * (-0.5f * 1.44269504f));
    const float t = __builtin_amdgcn_rcpf(fmaf(x, 0.325f, 1.f));
    float p = fmaf(t, 0.03382433f, -0.1135416f);
    p = fmaf(t, p, 0.08533306f);
    p = fmaf(t, p, 0.026032995f);
    p = fmaf(t, p, 0.09351984f);
    p = fmaf(t, p, 0.11550343f);
    p = fmaf(t, p, 0.12967211f);
    p = fmaf(t, p, 0.12965615f);
    tail = t * p * r.e;
  }
  r.cdf = z < 0.f ? tail : 1.f - tail;
  return r;
}
// act(z) of the ungated projection, and its derivative.
template <typename T, int W> __device__ __forceinline__ void activate_all(float (&z)[W], int act) {
  if (act == ACT_SILU) {
#pragma unroll
    for (int j = 0; j < W; ++j) z[j] *= sigmoid_for<T>(z[j]);
  } else if (act == ACT_GELU) {
#pragma unroll
    for (int j = 0; j < W; ++j) z[j] *= normal<T>(z[j]).cdf;
  }
}
// (slopes: of the two activations; without one dz is dy)
template <typename T, int W> __device__ __forceinline__ void slope_all(float (&z)[W], int act) {
  if (act == ACT_SILU) {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const float s = sigmoid_for<T>(z[j]);
      z[j] = s * (1.f + z[j] * (1.f - s));
    }
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const Normal r = normal<T>(z[j]);
      z[j] = fmaf(z[j] * 0.398942280f, r.e, r.cdf);
    }
  }
}
// For 16-bit results both tanh and the sigmoid come from exponentials of at most 1 and one reciprocal:
//   tanh(|g| / b1) = (1 - a) / (1 + a), a = exp(-2 |g| / b1);  sigmoid(|g|) = 1 / (1 + b), b = exp(-|g|)
// and where 1 - a cancels, tanh from a polynomial (relative error 2^-23 below 0.1).  The other factor's tanh is a polynomial
// below 0.6 (2^-22), where all of a wave's values are in nearly every epilogue.
struct Parts {
  float a, b, num, den;  // tanh = num / (1 + a), den = (1 + a) (1 + b)
};
__device__ __forceinline__ Parts gate_parts(float g, const Gate& c) {
  constexpr float kLog2e = 1.44269504f;
  Parts r;
  const float x = fabsf(g) * c.i1, x2 = x * x;
  r.a = __builtin_amdgcn_exp2f(x * (-2.f * kLog2e));
  r.b = __builtin_amdgcn_exp2f(fabsf(g) * -kLog2e);
  float near = x * (0.999999998f + x2 * (-0.333330316f + x2 * 0.132527533f)), far = 1.f - r.a;
  near = fmaf(near, r.a, near);
  // both are formed, one is taken: the compiler would make a branch of it for every value (52 us for 49, 8192 x 1024 x 2048 in
  // e4m3)
  asm volatile("" : "+v"(near), "+v"(far));
  r.num = x2 < 0.01f ? near : far;
  const float t = 1.f + r.b;
  r.den = fmaf(r.a, t, t);
  return r;
}
__device__ __forceinline__ float tanh_below(float x) {
  const float x2 = x * x;
  return x * (0.999999927f + x2 * (-0.333323102f + x2 * (0.133101752f + x2 * (-0.0521015118f + x2 * 0.0154754365f))));
}
__device__ __forceinline__ float tanh_any(float x) {
  const float e = __builtin_amdgcn_exp2f(fabsf(x) * (-2.f * 1.44269504f));
  const float far = copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e), x);
  return x * x < 0.36f ? tanh_below(x) : far;
}
// tanh(u / b2) of W values
template <typename T, int W> __device__ __forceinline__ void tanh_all(const float (&u)[W], float scale, float (&t)[W]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < W; ++j) t[j] = tanhf(u[j] * scale);
    return;
  }
  bool below = true;
#pragma unroll
  for (int j = 0; j < W; ++j) {
    t[j] = u[j] * scale;
    below = below && fabsf(t[j]) < 0.6f;
  }
  if (__all(below)) {
#pragma unroll
    for (int j = 0; j < W; ++j) t[j] = tanh_below(t[j]);
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) t[j] = tanh_any(t[j]);
  }
}
// The same with the slopes 1 - tanh^2 = 4 e / (1 + e)^2, e = exp(-2 |x|): the difference loses what the slope is once tanh is near 1
// (a twentieth of it at x = 8, all of it beyond 9.02).
__device__ __forceinline__ float sech2(float e, float inverse) { return 4.f * e * inverse * inverse; }
template <typename T, int W> __device__ __forceinline__ void tanh_slopes_all(const float (&u)[W], float scale, float (&t)[W], float (&d)[W]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const float x = u[j] * scale, e = expf(-2.f * fabsf(x));
      t[j] = tanhf(x), d[j] = sech2(e, 1.f / (1.f + e));
    }
    return;
  }
  bool below = true;
#pragma unroll
  for (int j = 0; j < W; ++j) {
    t[j] = u[j] * scale;
    below = below && fabsf(t[j]) < 0.6f;
  }
  if (__all(below)) {
#pragma unroll
    for (int j = 0; j < W; ++j) t[j] = tanh_below(t[j]), d[j] = 1.f - t[j] * t[j];
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const float e = __builtin_amdgcn_exp2f(fabsf(t[j]) * (-2.f * 1.44269504f)), r = __builtin_amdgcn_rcpf(1.f + e);
      d[j] = sech2(e, r);
      t[j] = t[j] * t[j] < 0.36f ? tanh_below(t[j]) : copysignf((1.f - e) * r, t[j]);
    }
  }
}
// g = a(g) b(u)
template <typename T, int W> __device__ __forceinline__ void gated(float (&g)[W], const float (&u)[W], const Gate& c) {
  if (c.act == ACT_SILU) {
#pragma unroll
    for (int j = 0; j < W; ++j) g[j] = g[j] * sigmoid_for<T>(g[j]) * u[j];
    return;
  }
  float t[W];
  tanh_all<T, W>(u, c.i2, t);
#pragma unroll
  for (int j = 0; j < W; ++j) {
    if constexpr (sizeof(T) == 4) {
      g[j] = c.b1 * tanhf(g[j] * c.i1) * sigmoid_for<T>(g[j]) * (c.b2 * t[j]);
    } else {
      const Parts r = gate_parts(g[j], c);
      const float s = g[j] < 0.f ? -r.b : 1.f;  // the sign, and sigmoid(g) = b / (1 + b) below 0
      // each tanh beside its own beta: b1 b2 may be 2^128
      g[j] = r.num * s * __builtin_amdgcn_rcpf(r.den) * c.b1 * (c.b2 * t[j]);
    }
  }
}
// g, u = dh a'(g) b(u), dh a(g) b'(u)
template <typename T, int W>
__device__ __forceinline__ void gated_slopes(float (&g)[W], float (&u)[W], const float (&dh)[W], const Gate& c) {
  if (c.act == ACT_SILU) {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const float s = sigmoid_for<T>(g[j]), a = g[j] * s;
      g[j] = dh[j] * u[j] * (s + a * (1.f - s));
      u[j] = dh[j] * a;
    }
    return;
  }
  float t2[W], d2[W];
  tanh_slopes_all<T, W>(u, c.i2, t2, d2);
#pragma unroll
  for (int j = 0; j < W; ++j) {
    float s, ns, t1, d1;  // sigmoid(g), sigmoid(-g), tanh and its slope
    if constexpr (sizeof(T) == 4) {
      const float x = g[j] * c.i1, e = expf(-2.f * fabsf(x));
      s = sigmoid_for<T>(g[j]), ns = sigmoid_for<T>(-g[j]), t1 = tanhf(x), d1 = sech2(e, 1.f / (1.f + e));
    } else {
      const Parts r = gate_parts(g[j], c);
      const float q = __builtin_amdgcn_rcpf(r.den), big = fmaf(r.a, q, q), small = r.b * big;
      const float inverse = fmaf(r.b, q, q);  // 1 / (1 + a)
      t1 = copysignf(r.num * inverse, g[j]), d1 = sech2(r.a, inverse);
      s = g[j] < 0.f ? small : big, ns = g[j] < 0.f ? big : small;
    }
    const float a = c.b1 * t1 * s;
    g[j] = dh[j] * (c.b2 * t2[j]) * (s * d1 + a * ns);
    u[j] = dh[j] * a * d2[j];
  }
}

// W consecutive elements of a row from column n, zeros from `n_end` on.  Rows start anywhere: the hardware takes vectors at any
// address.  FULL: none is beyond.
template <typename T, int W, bool FULL = false> __device__ __forceinline__ void load_cols(const T* row, int n, int n_end, float (&x)[W]) {
  if (FULL || n + W <= n_end) {
    T v[W];
    __builtin_memcpy(v, row + n, sizeof(v));
#pragma unroll
    for (int j = 0; j < W; ++j) x[j] = io<T>::to_f32(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) x[j] = n + j < n_end ? io<T>::load(row, n + j) : 0.f;
  }
}
template <typename T, int W, bool FULL = false> __device__ __forceinline__ void store_cols(T* row, int n, int n_end, const float (&x)[W]) {
  typedef typename native<T>::type N;
  N v[W];
#pragma unroll
  for (int j = 0; j < W; ++j) v[j] = static_cast<N>(x[j]);
  if (FULL || n + W <= n_end) {
    __builtin_memcpy(row + n, v, sizeof(v));
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j)
      if (n + j < n_end) __builtin_memcpy(row + n + j, v + j, sizeof(T));
  }
}

// The fp32 sums that a forward kept, read once.  (Written with ordinary stores: nontemporal ones of a lane's 16 bytes, a part of
// a line each, took the forward and backward of 8192 x 4096 x 8192 from 2531 to 2709 us.)
typedef f32x4 f32x4_any __attribute__((aligned(4)));
template <int W, bool FULL> __device__ __forceinline__ void kept_cols(const float* row, int n, int n_end, float (&x)[W]) {
  if (FULL || n + W <= n_end) {
#pragma unroll
    for (int j = 0; j < W; j += 4) {
      const f32x4 v = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any*>(row + n + j));
#pragma unroll
      for (int i = 0; i < 4; ++i) x[j + i] = v[i];
    }
  } else {
    load_cols<float, W, FULL>(row, n, n_end, x);
  }
}

// What the epilogue needs of W consecutive columns from n, for all of a lane's rows.
template <int W> struct Columns {
  float ws[W], ws2[W], bias[W];
};
template <typename E, typename T, int KIND, int W, bool FULL = false> __device__ __forceinline__ Columns<W> columns_at(const Args& p, int n) {
  Columns<W> c = {};
  if constexpr (sizeof(E) == 1) {
    load_cols<float, W, FULL>(p.ws, n, p.n, c.ws);
    if constexpr (KIND == GATED) load_cols<float, W, FULL>(p.ws2, n, p.n, c.ws2);
  }
  if constexpr (KIND == LINEAR || KIND == LINEAR_DZ)
    if (p.bias != nullptr) load_cols<T, W, FULL>(static_cast<const T*>(p.bias), n, p.n, c.bias);
  return c;
}

// z ws xs.  A sum z of products of e4m3 values is 0 or 2^-18 to 2^48, so z times an ordinary weight's scale, from 2^-100 to 2^70, is a
// normal number, and the result is rounded as itself for any xs.  (z times xs ws, which may be infinite, would lose a z of 0.)  FAR: of
// other columns (a weight's row of zeros has the scale 2^-126) the powers of two are added and come last.  Asked once for a lane's
// columns; for each of its rows that costs 7 us of 46 (e4m3 8192 x 1024 x 2 x 2048).
template <int W> __device__ __forceinline__ bool far_scale(const float (&ws)[W]) {
  float low = __builtin_inff(), high = 0.f;
#pragma unroll
  for (int j = 0; j < W; ++j) low = fminf(low, fabsf(ws[j])), high = fmaxf(high, fabsf(ws[j]));
  return !(low >= 0x1p-100f && high <= 0x1p70f);
}
template <bool FAR, int W> __device__ __forceinline__ void scale_all(float (&z)[W], float xs, const float (&ws)[W]) {
#pragma unroll
  for (int j = 0; j < W; ++j) {
    if constexpr (FAR)
      z[j] = ldexpf(z[j] * __builtin_amdgcn_frexp_mantf(ws[j]) * __builtin_amdgcn_frexp_mantf(xs),
                    __builtin_amdgcn_frexp_expf(ws[j]) + __builtin_amdgcn_frexp_expf(xs));
    else
      z[j] = z[j] * ws[j] * xs;
  }
}

// The lane's columns of one row of one product (two for the gated kinds), W consecutive ones from n.
// other: the row's residual (dy, dh) where the caller has read it.
template <typename E, typename T, int KIND, int W, bool FULL = false, bool FAR = sizeof(E) == 1>
__device__ __forceinline__ void finish(const Args& p, int m, int n, const Columns<W>& c, float (&z)[W], float (&z2)[W], float xs, int split,
                                       const float* other = nullptr) {
  if constexpr (sizeof(E) == 1) {
    scale_all<FAR, W>(z, xs, c.ws);
    if constexpr (KIND == GATED) scale_all<FAR, W>(z2, xs, c.ws2);
  }
  if constexpr (KIND == LINEAR || KIND == LINEAR_DZ) {
    float t[W];
    if (p.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < W; ++j) z[j] += c.bias[j];
    }
    if constexpr (KIND == LINEAR) {
      if (p.keep != nullptr) store_cols<float, W, FULL>(p.keep + static_cast<int64_t>(m) * p.n, n, p.n, z);
      activate_all<T, W>(z, p.act);
      if (p.other != nullptr) {
        if (other == nullptr) load_cols<T, W, FULL>(static_cast<const T*>(p.other) + m * p.ldother, n, p.n, t);
#pragma unroll
        for (int j = 0; j < W; ++j) z[j] += other != nullptr ? other[j] : t[j];
      }
      store_cols<T, W, FULL>(static_cast<T*>(p.out) + m * p.ldo, n, p.n, z);
    } else {
      load_cols<T, W, FULL>(static_cast<const T*>(p.other) + m * p.ldother, n, p.n, t);
      slope_all<T, W>(z, p.act);
      // up to the row's end: the columns past the last are read as the contraction's of a later product
#pragma unroll
      for (int j = 0; j < W; ++j) z[j] = FULL || n + j < p.n ? t[j] * z[j] : 0.f;
      store_cols<T, W, FULL>(static_cast<T*>(p.out) + m * p.ldo, n, static_cast<int>(p.ldo), z);
    }
  } else if constexpr (KIND == GATED || KIND == GATED_DZ) {
    const Gate& gate = p.gate;
    if constexpr (KIND == GATED) {
      if (p.keep != nullptr) {
        float* row = p.keep + static_cast<int64_t>(m) * 2 * p.n;
        store_cols<float, W, FULL>(row, n, p.n, z);
        store_cols<float, W, FULL>(row + p.n, n, p.n, z2);
      }
      gated<T, W>(z, z2, gate);
      store_cols<T, W, FULL>(static_cast<T*>(p.out) + m * p.ldo, n, p.n, z);
    } else {
      float dh[W];
      load_cols<T, W, FULL>(static_cast<const T*>(p.other) + m * p.ldother, n, p.n, dh);
      gated_slopes<T, W>(z, z2, dh, gate);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        z[j] = FULL || n + j < p.n ? z[j] : 0.f;
        z2[j] = FULL || n + j < p.n ? z2[j] : 0.f;
      }
      T* row = static_cast<T*>(p.out) + m * p.ldo;
      store_cols<T, W, FULL>(row, n, static_cast<int>(p.second), z);
      store_cols<T, W, FULL>(row + p.second, n, static_cast<int>(p.second), z2);
    }
  } else if constexpr (KIND == DX) {
    store_cols<T, W, FULL>(static_cast<T*>(p.out) + m * p.ldo, n, p.n, z);
  } else {
    const int s = m / p.seg, r = m - s * p.seg;
    if (r >= p.seg_valid) return;
    const int64_t row = static_cast<int64_t>(s) * p.seg_valid + r;
    if (p.partial != nullptr)
      store_cols<float, W, FULL>(p.partial + (static_cast<int64_t>(split) * (p.m / p.seg) * p.seg_valid + row) * p.n, n, p.n, z);
    else
      store_cols<T, W, FULL>(static_cast<T*>(p.out) + row * p.ldo, n, p.n, z);
  }
}

// f of the result's type: the operands', or for 8-bit ones that of the call.
template <typename E, typename F> __device__ __forceinline__ void by_result(const Args& p, F&& f) {
  if constexpr (sizeof(E) == 1) {
    if (p.out_dtype == VMI_F32) f(float{});
    else if (p.out_dtype == VMI_BF16) f(bf16_t{});
    else f(f16_t{});
  } else {
    f(typename memory<E>::type{});
  }
}

template <typename E, int KIND, typename S, int GROUPS>
__global__ __launch_bounds__(S::THREADS * GROUPS, S::THREADS == 512 && S::STAGE > 40960 ? 2 : 4) void product_kernel(Args p) {
  constexpr bool AMN = KIND == DW, BMN = KIND == DX || KIND == DW, PERM = !BMN;
  constexpr bool PAIR = KIND == GATED || KIND == GATED_DZ;
  constexpr int SIZE = sizeof(E), KT = 128 / SIZE, TN = PAIR ? S::HN : 2 * S::HN;
  __shared__ __align__(1024) char lds[GROUPS * 2 * S::STAGE];
  int block = blockIdx.x, split = 0;
  if constexpr (KIND == DW) {
    split = block / (p.tiles_m * p.tiles_n);
    block -= split * (p.tiles_m * p.tiles_n);
  }
  int tm, tn;
  tile_of(block, p.tiles_m, p.tiles_n, p.group, tm, tn);
  const int m0 = tm * 2 * S::HM, n0 = tn * TN;
  Operands o;
  o.lda = static_cast<unsigned>(p.lda * SIZE), o.ldb = static_cast<unsigned>(p.ldb * SIZE);
  o.a_step = AMN ? KT * p.lda * SIZE : 128, o.b_step = BMN ? KT * p.ldb * SIZE : 128;
  o.k = p.k;
  int64_t k0 = 0;
  if constexpr (KIND == DW) {
    k0 = static_cast<int64_t>(split) * p.split_k;
    o.k = p.k - static_cast<int>(k0) < p.split_k ? p.k - static_cast<int>(k0) : p.split_k;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int m = m0 + h * S::HM, n = PAIR ? n0 : n0 + h * S::HN;
    const char* a = static_cast<const char*>(p.a) + (AMN ? k0 * p.lda + m : m * p.lda) * SIZE;
    o.a[h] = a;
    o.a2[h] = a + p.second * SIZE;
    o.a_inside[h] = p.m - m;
    const char* b = static_cast<const char*>(PAIR && h == 1 ? p.b2 : p.b);
    o.b[h] = b + (BMN ? k0 * p.ldb + n : n * p.ldb) * SIZE;
    o.b2[h] = static_cast<const char*>(p.b2) + static_cast<int64_t>(n) * SIZE;
    o.b_inside[h] = p.n - n;
  }
  Acc<S> acc;
  if (KIND == DX && p.b2 != nullptr)
    tile_product<E, AMN, BMN, S, KIND == DX ? 2 : 1, GROUPS>(o, lds, acc);
  else
    tile_product<E, AMN, BMN, S, 1, GROUPS>(o, lds, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x % S::THREADS >> 6, wm = wave / S::WN, wn = wave % S::WN;
  // the parts of the tile that a thread finishes
  constexpr int HMS = GROUPS > 1 ? 1 : 2, HNS = PAIR || GROUPS < 4 ? 2 : 1;
  int hm0 = 0, hn0 = 0;
  if constexpr (GROUPS > 1) {
    join_groups<S, GROUPS, HNS>(lds, acc);
    const int group = threadIdx.x / S::THREADS;
    if (PAIR && group >= 2) return;
    hm0 = group & 1, hn0 = HNS == 1 ? group >> 1 : 0;
  }
  constexpr bool SWAP = !PERM && S::NF == 2;
  constexpr int W = PERM ? 4 * S::NF : SWAP ? 8 : 4, PARTS = PERM || SWAP ? 1 : S::NF;
  // (C's columns 16 j + 4 g .. of lane group g) to 8 consecutive ones: groups 2 i and 2 i + 1 exchange one of their two fours,
  // after which group g holds 8 columns of fragment g % 2.
  if constexpr (SWAP) {
#pragma unroll
    for (int hm = 0; hm < HMS; ++hm)
#pragma unroll
      for (int hn = 0; hn < HNS; ++hn)
#pragma unroll
        for (int f = 0; f < S::MF; ++f)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            f32x4 &lo = acc.v[hm][hn][f][0], &hi = acc.v[hm][hn][f][1];
            const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(lo[r]), __float_as_uint(hi[r]), false, false);
            lo[r] = __uint_as_float(x[0]), hi[r] = __uint_as_float(x[1]);
          }
  }
  auto write = [&](auto tag, auto full) {
    using T = decltype(tag);
    constexpr bool FULL = decltype(full)::value;
#pragma unroll
    for (int hn = 0; hn < (PAIR ? 1 : HNS); ++hn)
#pragma unroll
      for (int q = 0; q < PARTS; ++q) {
        const int g = lane >> 4;
        const int n = n0 + (hn0 + hn) * S::HN + (SWAP ? wn * 32 + (g & 1) * 16 + (g >> 1) * 8 : column_of<S, PERM>(wn, lane, q));
        const Columns<W> cols = columns_at<E, T, KIND, W, FULL>(p, n);
        auto rows = [&](auto far) {
#pragma unroll
          for (int hm = 0; hm < HMS; ++hm)
#pragma unroll
            for (int f = 0; f < S::MF; ++f) {
              const int m = m0 + (hm0 + hm) * S::HM + wm * 16 * S::MF + f * 16 + (lane & 15);
              if (!FULL && m >= p.m) continue;
              float z[W], z2[W];
#pragma unroll
              for (int j = 0; j < W; ++j) {
                z[j] = acc.v[hm][hn][f][PERM || SWAP ? j / 4 : q][j % 4];
                z2[j] = PAIR ? acc.v[hm][1][f][PERM ? j / 4 : q][j % 4] : 0.f;
              }
              finish<E, T, KIND, W, FULL, decltype(far)::value>(p, m, n, cols, z, z2, SIZE == 1 ? p.xs[m] : 1.f, split);
            }
        };
        if constexpr (SIZE == 1 && !FULL) rows(std::true_type{});
        else if (SIZE == 1 && __any(far_scale<W>(cols.ws) || (PAIR && far_scale<W>(cols.ws2)))) rows(std::true_type{});
        else rows(std::false_type{});
      }
  };
  // most tiles lie inside the result: their accesses need no conditions, which would keep them from being in flight together
  if (m0 + 2 * S::HM <= p.m && n0 + TN <= p.n)
    by_result<E>(p, [&](auto tag) { write(tag, std::true_type{}); });
  else
    by_result<E>(p, [&](auto tag) { write(tag, std::false_type{}); });
}

typedef Shape<128, 128, 2, 4> Large;
typedef Shape<128, 64, 4, 2> Tall;
typedef Shape<64, 64, 4, 2> Middle;
typedef Shape<32, 32, 2, 2> Small;

// kind over operands of one type (feed_forward_*.hip).
int product_bf16(Kind kind, Args p, hipStream_t stream);
int product_f16(Kind kind, Args p, hipStream_t stream);
int product_f32(Kind kind, Args p, hipStream_t stream);
int product_e4m3(Kind kind, Args p, hipStream_t stream);

// Rows of tiles in a column of tile_of: the tiles that an XCD's 32 compute units have at a time then cover about as many rows of
// the result as columns, and read the fewest of the operands' rows into its L2.  dW of 2048 x 1024 over 8192 rows, 64 tiles of 256
// x 128 in four shares, in us: columns of 1 44.7, of 2 45.6, of 4 46.0, of 8 54.8 (all of one operand in every L2).
template <typename S> int rows_of_tiles(int64_t tiles, int concurrent) {
  int64_t run = (tiles + 7) / 8;
  if (run > 32 * concurrent) run = 32 * concurrent;
  int g = 1;
  while (2 * g * g * S::HM <= run * S::HN) g *= 2;
  return g;
}

template <typename E, int KIND, typename S, int GROUPS = 1> int launch_product(Args p, hipStream_t stream) {
  constexpr bool PAIR = KIND == GATED || KIND == GATED_DZ;
  const int tn = PAIR ? S::HN : 2 * S::HN;
  const int64_t tiles_m = (static_cast<int64_t>(p.m) + 2 * S::HM - 1) / (2 * S::HM), tiles_n = (static_cast<int64_t>(p.n) + tn - 1) / tn;
  const int64_t blocks = tiles_m * tiles_n * (KIND == DW ? p.splits : 1);
  if (blocks == 0) return VMI_OK;
  if (!grid_fits(blocks, S::THREADS * GROUPS)) return VMI_ERR_UNSUPPORTED;
  p.tiles_m = static_cast<int>(tiles_m), p.tiles_n = static_cast<int>(tiles_n);
  p.group = rows_of_tiles<S>(tiles_m * tiles_n, S::STAGE > 40960 || GROUPS > 1 ? 1 : 65536 / S::STAGE);
  hipLaunchKernelGGL((product_kernel<E, KIND, S, GROUPS>), dim3(static_cast<unsigned>(blocks)), dim3(S::THREADS * GROUPS), 0, stream, p);
  return hip_status(hipGetLastError());
}

inline int64_t tiles(int64_t m, int64_t n, int tm, int tn) { return ((m + tm - 1) / tm) * ((n + tn - 1) / tn); }

// What the tiles of a shape take, in units of their own: rounds of one tile for each of the 256 compute units (two tiles of 128 x 128
// or four of 64 x 64 in one at a time count alike), by what a round took in relation to one of 256 x 256 tiles.  A last round that
// leaves compute units idle is shorter: under the power limit (16 bits) the others' clocks rise.  In fp32 the matrix cores bound every
// tile, and a round is its tile's elements.
//
// us of 256 x 256, 256 x 128, 128 x 128, 64 x 64, rows x k x columns; bf16: 8192 x 1024 x 2048 (256 of the largest tiles) 30.5 33.9
// 34.9 51.8, 4352 x 1024 x 2048 (136) 27.4 30.3 27.1 31.6, 4352 x 2048 x 1024 (68) 37.0 24.5 28.1 33.3, 2048 x 1024 x 2048 (64) 22.8
// 15.1 12.0 14.7, 1024 x 1024 x 2048 (32) 22.0 13.7 10.9 9.1; e4m3: 4352 x 1024 x 2048 20.4 22.2 18.9 21.8, 9000 x 1024 x 2304 36.2
// 36.2 30.2 46.2; fp32: 8192 x 4096 x 4096 1874 1910 1901 2017, 2048 x 2048 x 2048 470 244 133 134, 1787 x 3840 x 3228 874 450 445
// 356, 2500 x 700 x 900 171 89 50 39.
struct Rounds {
  int size;  // an operand's element
  int64_t time(int64_t tiles, int shape) const {
    constexpr int weight[3][4] = {{1000, 565, 300, 130}, {1000, 565, 310, 130}, {1000, 510, 255, 67}};
    if (!grid_fits(tiles, shape == 3 ? Small::THREADS : Large::THREADS)) return INT64_MAX;
    const int least = size == 4 ? 256 : size == 2 ? 192 : 230;  // of 256, what a round with one tile takes
    const int64_t rest = tiles % 256;
    return (tiles / 256 * 256 + (rest == 0 ? 0 : least + (256 - least) * rest / 256)) * weight[size / 2][shape];
  }
};

// What a product runs as: a tile (the last: four groups of its waves share the contraction), or the kernel for a few rows, 16, 32 or 64
// of them a workgroup.
enum Form { LARGE, TALL, MIDDLE, SMALL, SMALL_BY_FOUR, ROWS_16, ROWS_32, ROWS_64 };

// The kernel for a few rows takes a result of up to 512 fragments of 16 x 16 (fp32: 1536, and 2048 of the gated form), and any of up
// to 16 rows that a grid's threads hold.  Both sides in us, rows / tiles: bf16 K 2048 N 1024 M 128 7.7 / 9.1, M 256 11.5 / 9.2; bf16
// K 1024 N 4096 M 32 5.7 / 6.2, M 64 8.4 / 6.4; e4m3 K 4096 N 4096 M 32 8.1 / 9.0, M 64 12.1 / 9.0; fp32 K 2048 N 1024 M 256 22 / 37,
// M 384 39 / 38; fp32 K 4096 N 4096 M 96 64 / 69, M 128 74 / 72, gated (F 2048) M 128 53 / 71.
inline bool few_rows(Kind kind, int size, const Args& p) {
  const int64_t cols = kind == GATED ? 2 * static_cast<int64_t>(p.n) : p.n;
  if ((kind != LINEAR && kind != GATED) || !grid_fits((static_cast<int64_t>(p.n) + 15) / 16, 512)) return false;
  return p.m <= 16 || tiles(p.m, cols, 16, 16) <= (size < 4 ? 512 : kind == GATED ? 2048 : 1536);
}
// Rows are split over workgroups too while there are fewer of those than compute units: a workgroup's x and weights both go
// through its compute unit (64 rows, K 2048, N 1024 in fp16: 16 rows a workgroup 6.6 us, 64 12.3).  A gated result of 512 fragments
// has at most 85 columns of them with more than 32 rows, which never need workgroups of 64.
inline Form rows_form(Kind kind, int size, const Args& p) {
  const int64_t cols = (static_cast<int64_t>(p.n) + 15) / 16;
  int mt = p.m <= 16 ? 1 : p.m <= 32 || (kind == GATED && size < 4) ? 2 : 4;
  while (mt > 1 && cols * ((p.m + 16 * mt - 1) / (16 * mt)) <= 128) mt /= 2;
  return mt == 1 ? ROWS_16 : mt == 2 ? ROWS_32 : ROWS_64;
}

inline Form form_of(Kind kind, int size, const Args& p) {
  if (few_rows(kind, size, p)) return rows_form(kind, size, p);
  const bool pair = kind == GATED || kind == GATED_DZ;
  const int64_t cols = pair ? 2 * static_cast<int64_t>(p.n) : p.n;
  const int64_t shares = kind == DW ? p.splits : 1;
  // With a short contraction SiTU's epilogue costs as much as the products: of two workgroups a compute unit one multiplies meanwhile.
  // us with tiles of 128 x 128 / of 256 x 256, 8192 rows, F 2048, on one card: e4m3 K 512 35.4 / 40.6, K 1024 49.1 / 50.7, K 1536 61.3 /
  // 61.0; bf16 K 512 47.2 / 46.4, K 1024 71.3 / 66.6.
  if (const int64_t t = tiles(p.m, cols, 128, 128);
      pair && p.gate.act == ACT_SITU && p.k <= 8 * (128 / size) && t >= 160 && grid_fits(t, Middle::THREADS))
    return MIDDLE;
  const Rounds r = {size};
  const int64_t l = r.time(tiles(p.m, cols, 256, 256) * shares, 0), t = r.time(tiles(p.m, cols, 256, 128) * shares, 1);
  const int64_t m = r.time(tiles(p.m, cols, 128, 128) * shares, 2), s = r.time(tiles(p.m, cols, 64, 64) * shares, 3);
  if (l <= t && l <= m && l <= s) return LARGE;
  if (t <= m && t <= s) return TALL;
  if (m <= s) return MIDDLE;
  // Four groups of a tile's waves share a long contraction where the tiles leave compute units idle or at one workgroup: a step's
  // latency, not its data, bounds them.  us with four / one (rows x k x columns): bf16 512 x 4096 x 512 15.5 / 21.7, 256 x 4096 x
  // 4096 16.6 / 22.8, 1024 x 1024 x 1024 (16 steps) 7.8 / 6.9, 384 x 4096 x 4096 (384 tiles) 29.7 / 25.2; fp32 777 x 1000 x 1037
  // 22.7 / 24.2, 256 x 4096 x 4096 70 / 86; e4m3 256 x 4096 x 4096 10.0 / 10.4.  The other kinds have short contractions: DW's
  // shares, and dz where the forward kept no sums.
  const bool groups = (kind == LINEAR || kind == GATED || kind == DX) && tiles(p.m, cols, 64, 64) <= 256 && p.k > 31 * (128 / size);
  return groups ? SMALL_BY_FOUR : SMALL;
}

template <typename E, int KIND, int MT> int launch_rows(const Args& p, hipStream_t stream);  // feed_forward_rows.h

template <typename E, int KIND> int product_of_kind(const Args& p, hipStream_t stream) {
  const Form form = form_of(static_cast<Kind>(KIND), sizeof(E), p);
  if constexpr (KIND == LINEAR || KIND == GATED) {
    if (form == ROWS_16) return launch_rows<E, KIND, 1>(p, stream);
    if (form == ROWS_32) return launch_rows<E, KIND, 2>(p, stream);
    if constexpr (KIND == LINEAR || sizeof(E) == 4)
      if (form == ROWS_64) return launch_rows<E, KIND, 4>(p, stream);
  }
  if constexpr (KIND == LINEAR || KIND == GATED || KIND == DX)
    if (form == SMALL_BY_FOUR) return launch_product<E, KIND, Small, 4>(p, stream);
  switch (form) {
    case LARGE: return launch_product<E, KIND, Large>(p, stream);
    case TALL: return launch_product<E, KIND, Tall>(p, stream);
    case MIDDLE: return launch_product<E, KIND, Middle>(p, stream);
    default: return launch_product<E, KIND, Small>(p, stream);
  }
}

template <typename E> int product_of(Kind kind, const Args& p, hipStream_t stream) {
  switch (kind) {
    case LINEAR: return product_of_kind<E, LINEAR>(p, stream);
    case GATED: return product_of_kind<E, GATED>(p, stream);
    default: break;
  }
  if constexpr (sizeof(E) > 1) {
    switch (kind) {
      case LINEAR_DZ: return product_of_kind<E, LINEAR_DZ>(p, stream);
      case GATED_DZ: return product_of_kind<E, GATED_DZ>(p, stream);
      case DX: return product_of_kind<E, DX>(p, stream);
      case DW: return product_of_kind<E, DW>(p, stream);
      default: break;
    }
  }
  return VMI_ERR_INVALID_ARG;
}

}  // namespace prod
}  // namespace vmi
