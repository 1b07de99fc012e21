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

struct Args {
  const void* a;     // x, dz
  const void* b;     // the weight, x
  const void* b2;    // the second weight
  int64_t lda, ldb, ldb2;  // elements
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
  int seg, seg_valid;      // DW: rows of the result come in segments of seg, of which seg_valid are stored
  int act;
  float beta1, beta2;
  int vec;                 // rows of out and other are whole 16-byte pieces
};

template <typename E> struct memory { typedef E type; };
template <> struct memory<__bf16> { typedef bf16_t type; };

// act(z) and its derivative of the ungated projection.
template <typename T> __device__ __forceinline__ float activate(float z, int act) {
  if (act == ACT_SILU) return z * sigmoid_for<T>(z);
  if (act == ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.707106781f));
  return z;
}
template <typename T> __device__ __forceinline__ float slope(float z, int act) {
  if (act == ACT_SILU) {
    const float s = sigmoid_for<T>(z);
    return s * (1.f + z * (1.f - s));
  }
  if (act == ACT_GELU) {
    const float e = sizeof(T) == 4 ? expf(-0.5f * z * z) : __expf(-0.5f * z * z);
    return 0.5f * (1.f + erff(z * 0.707106781f)) + z * 0.398942280f * e;
  }
  return 1.f;
}
struct Gate {
  int act;
  float b1, b2, i1, i2;
};
// The parts of tanh(x) = sign(x) num / den: (1 - e) / (1 + e) with e = exp(-2|x|), and near 0, where 1 - e cancels, a polynomial
// (the next term is below 2^-24 of it) over 1.
template <typename T> __device__ __forceinline__ void tanh_parts(float x, float& num, float& den) {
  const float a = fabsf(x), x2 = x * x;
  const float e = __expf(-2.f * a);
  const float near = a + a * x2 * (-0.333333333f + x2 * (0.133333333f + x2 * -0.0539682540f));
  num = x2 < 0.01f ? near : 1.f - e;
  den = x2 < 0.01f ? 1.f : 1.f + e;
}
// a(g) b(u).  16-bit results: the quotients of the two tanh and the sigmoid over one reciprocal, their exponentials at most 1.
template <typename T> __device__ __forceinline__ float gated(float g, float u, const Gate& c) {
  if (c.act == ACT_SILU) return g * sigmoid_for<T>(g) * u;
  if constexpr (sizeof(T) == 4) return c.b1 * tanhf(g * c.i1) * sigmoid_for<T>(g) * (c.b2 * tanhf(u * c.i2));
  float n1, d1, n2, d2;
  tanh_parts<T>(g * c.i1, n1, d1);
  tanh_parts<T>(u * c.i2, n2, d2);
  const float e = __expf(-fabsf(g)), s = g < 0.f ? e : 1.f;  // sigmoid(g) = s / (1 + e)
  const float h = c.b1 * c.b2 * n1 * n2 * s * __builtin_amdgcn_rcpf(d1 * d2 * (1.f + e));
  return (__float_as_uint(g) ^ __float_as_uint(u)) >> 31 ? -h : h;
}
template <typename T>
__device__ __forceinline__ void gated_slopes(float g, float u, float dh, const Gate& c, float& dg, float& du) {
  if (c.act == ACT_SILU) {
    const float s = sigmoid_for<T>(g);
    dg = dh * u * s * (1.f + g * (1.f - s));
    du = dh * g * s;
    return;
  }
  float s, ns, t1, t2;  // sigmoid(g) and sigmoid(-g)
  if constexpr (sizeof(T) == 4) {
    s = sigmoid_for<T>(g), ns = sigmoid_for<T>(-g);
    t1 = tanhf(g * c.i1), t2 = tanhf(u * c.i2);
  } else {
    float n1, d1, n2, d2;
    tanh_parts<T>(g * c.i1, n1, d1);
    tanh_parts<T>(u * c.i2, n2, d2);
    const float e = __expf(-fabsf(g)), d3 = 1.f + e, d12 = d1 * d2, r = __builtin_amdgcn_rcpf(d12 * d3);
    const float big = d12 * r, small = e * big;
    s = g < 0.f ? small : big, ns = g < 0.f ? big : small;
    t1 = copysignf(n1 * (d2 * d3) * r, g), t2 = copysignf(n2 * (d1 * d3) * r, u);
  }
  const float a = c.b1 * t1 * s;
  dg = dh * c.b2 * t2 * (s * (1.f - t1 * t1) + a * ns);
  du = dh * a * (1.f - t2 * t2);
}

// W consecutive elements of a row from column n, zeros from `n_end` on.
template <typename T, int W> __device__ __forceinline__ void load_cols(const T* row, int n, int n_end, bool vec, float (&x)[W]) {
  if (vec && n + W <= n_end) {
    typedef typename native<T>::type N;
    typedef N Piece __attribute__((ext_vector_type(W)));
    const Piece v = *reinterpret_cast<const Piece*>(row + n);
#pragma unroll
    for (int j = 0; j < W; ++j) x[j] = static_cast<float>(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) x[j] = n + j < n_end ? io<T>::load(row, n + j) : 0.f;
  }
}
template <typename T, int W> __device__ __forceinline__ void store_cols(T* row, int n, int n_end, bool vec, const float (&x)[W]) {
  if (vec && n + W <= n_end) {
    typedef typename native<T>::type N;
    typedef N Piece __attribute__((ext_vector_type(W)));
    Piece v;
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = static_cast<N>(x[j]);
    *reinterpret_cast<Piece*>(row + n) = v;
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j)
      if (n + j < n_end) io<T>::store(row, n + j, x[j]);
  }
}

// The lane's columns of one row of one product (two for the gated kinds), W consecutive ones from n.
template <typename E, typename T, int KIND, int W>
__device__ __forceinline__ void finish(const Args& p, int m, int n, float (&z)[W], float (&z2)[W], float xs, int split) {
  const bool vec = p.vec;
  if constexpr (KIND == LINEAR || KIND == LINEAR_DZ) {
    float t[W];
    if constexpr (sizeof(E) == 1) {
#pragma unroll
      for (int j = 0; j < W; ++j) z[j] *= xs * (n + j < p.n ? p.ws[n + j] : 0.f);
    }
    if (p.bias != nullptr) {
      load_cols<T, W>(static_cast<const T*>(p.bias), n, p.n, false, t);
#pragma unroll
      for (int j = 0; j < W; ++j) z[j] += t[j];
    }
    if constexpr (KIND == LINEAR) {
#pragma unroll
      for (int j = 0; j < W; ++j) z[j] = activate<T>(z[j], p.act);
      if (p.other != nullptr) {
        load_cols<T, W>(static_cast<const T*>(p.other) + m * p.ldother, n, p.n, vec, t);
#pragma unroll
        for (int j = 0; j < W; ++j) z[j] += t[j];
      }
      store_cols<T, W>(static_cast<T*>(p.out) + m * p.ldo, n, p.n, vec, z);
    } else {
      load_cols<T, W>(static_cast<const T*>(p.other) + m * p.ldother, n, p.n, vec, t);
      // up to the row's end: the columns past the last are read as the contraction's of a later product
#pragma unroll
      for (int j = 0; j < W; ++j) z[j] = n + j < p.n ? t[j] * slope<T>(z[j], p.act) : 0.f;
      store_cols<T, W>(static_cast<T*>(p.out) + m * p.ldo, n, static_cast<int>(p.ldo), vec, z);
    }
  } else if constexpr (KIND == GATED || KIND == GATED_DZ) {
    const Gate c{p.act, p.beta1, p.beta2, 1.f / p.beta1, 1.f / p.beta2};
    if constexpr (sizeof(E) == 1) {
#pragma unroll
      for (int j = 0; j < W; ++j) {
        z[j] *= xs * (n + j < p.n ? p.ws[n + j] : 0.f);
        z2[j] *= xs * (n + j < p.n ? p.ws2[n + j] : 0.f);
      }
    }
    if constexpr (KIND == GATED) {
#pragma unroll
      for (int j = 0; j < W; ++j) z[j] = gated<T>(z[j], z2[j], c);
      store_cols<T, W>(static_cast<T*>(p.out) + m * p.ldo, n, p.n, vec, z);
    } else {
      float dh[W];
      load_cols<T, W>(static_cast<const T*>(p.other) + m * p.ldother, n, p.n, vec, dh);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        float dg = 0.f, du = 0.f;
        if (n + j < p.n) gated_slopes<T>(z[j], z2[j], dh[j], c, dg, du);
        z[j] = dg;
        z2[j] = du;
      }
      T* row = static_cast<T*>(p.out) + m * p.ldo;
      store_cols<T, W>(row, n, static_cast<int>(p.second), vec, z);
      store_cols<T, W>(row + p.second, n, static_cast<int>(p.second), vec, z2);
    }
  } else if constexpr (KIND == DX) {
    store_cols<T, W>(static_cast<T*>(p.out) + m * p.ldo, n, p.n, vec, z);
  } else {
    const int s = m / p.seg, r = m - s * p.seg;
    if (r >= p.seg_valid) return;
    const int64_t row = static_cast<int64_t>(s) * p.seg_valid + r;
    if (p.partial != nullptr)
      store_cols<float, W>(p.partial + (static_cast<int64_t>(split) * (p.m / p.seg) * p.seg_valid + row) * p.n, n, p.n,
                           p.n % W == 0, z);
    else
      store_cols<T, W>(static_cast<T*>(p.out) + row * p.ldo, n, p.n, vec, z);
  }
}

template <typename E, int KIND, typename S> __global__ __launch_bounds__(S::THREADS, S::THREADS == 512 && S::STAGE > 40960 ? 2 : 4)
void product_kernel(Args p) {
  constexpr bool AMN = KIND == DW, BMN = KIND == DX || KIND == DW, PERM = !BMN;
  constexpr bool PAIR = KIND == GATED || KIND == GATED_DZ;
  constexpr int SIZE = sizeof(E), KT = 128 / SIZE, TN = PAIR ? S::HN : 2 * S::HN;
  __shared__ __align__(1024) char lds[2 * S::STAGE];
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
    tile_product<E, AMN, BMN, S, KIND == DX ? 2 : 1>(o, lds, acc);
  else
    tile_product<E, AMN, BMN, S, 1>(o, lds, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / S::WN, wn = wave % S::WN;
  constexpr int W = PERM ? 4 * S::NF : 4, PARTS = PERM ? 1 : S::NF;
  auto write = [&](auto tag) {
    using T = decltype(tag);
#pragma unroll
    for (int hm = 0; hm < 2; ++hm)
#pragma unroll
      for (int f = 0; f < S::MF; ++f) {
        const int m = m0 + hm * S::HM + wm * 16 * S::MF + f * 16 + (lane & 15);
        if (m >= p.m) continue;
        float xs = 1.f;
        if constexpr (SIZE == 1) xs = p.xs[m];
#pragma unroll
        for (int hn = 0; hn < (PAIR ? 1 : 2); ++hn)
#pragma unroll
          for (int q = 0; q < PARTS; ++q) {
            const int n = n0 + hn * S::HN + column_of<S, PERM>(wn, lane, q);
            float z[W], z2[W];
#pragma unroll
            for (int j = 0; j < W; ++j) {
              z[j] = acc.v[hm][hn][f][PERM ? j / 4 : q][j % 4];
              z2[j] = PAIR ? acc.v[hm][1][f][PERM ? j / 4 : q][j % 4] : 0.f;
            }
            finish<E, T, KIND, W>(p, m, n, z, z2, xs, split);
          }
      }
  };
  if constexpr (SIZE == 1) {
    if (p.out_dtype == VMI_F32) write(float{});
    else if (p.out_dtype == VMI_BF16) write(bf16_t{});
    else write(f16_t{});
  } else {
    write(typename memory<E>::type{});
  }
}

typedef Shape<128, 128, 2, 4> Large;
typedef Shape<128, 64, 2, 4> Tall;
typedef Shape<64, 64, 2, 4> Middle;
typedef Shape<32, 32, 2, 2> Small;

// kind over operands of one type (feed_forward_*.hip).
int product_bf16(Kind kind, Args p, hipStream_t stream);
int product_f16(Kind kind, Args p, hipStream_t stream);
int product_f32(Kind kind, Args p, hipStream_t stream);
int product_e4m3(Kind kind, Args p, hipStream_t stream);

template <typename E, int KIND, typename S> int launch_product(Args p, hipStream_t stream) {
  constexpr bool PAIR = KIND == GATED || KIND == GATED_DZ;
  const int tn = PAIR ? S::HN : 2 * S::HN;
  const int64_t tiles_m = (static_cast<int64_t>(p.m) + 2 * S::HM - 1) / (2 * S::HM), tiles_n = (static_cast<int64_t>(p.n) + tn - 1) / tn;
  const int64_t blocks = tiles_m * tiles_n * (KIND == DW ? p.splits : 1);
  if (blocks == 0) return VMI_OK;
  if (!grid_fits(blocks, S::THREADS)) return VMI_ERR_UNSUPPORTED;
  p.tiles_m = static_cast<int>(tiles_m), p.tiles_n = static_cast<int>(tiles_n), p.group = 8;
  hipLaunchKernelGGL((product_kernel<E, KIND, S>), dim3(static_cast<unsigned>(blocks)), dim3(S::THREADS), 0, stream, p);
  return hip_status(hipGetLastError());
}

inline int64_t tiles(int64_t m, int64_t n, int tm, int tn) { return ((m + tm - 1) / tm) * ((n + tn - 1) / tn); }

template <typename E, int KIND> int product_of_kind(const Args& p, hipStream_t stream) {
  constexpr bool PAIR = KIND == GATED || KIND == GATED_DZ;
  const int64_t cols = PAIR ? 2 * static_cast<int64_t>(p.n) : p.n;
  const int64_t shares = KIND == DW ? p.splits : 1;
  if (tiles(p.m, cols, 256, 256) * shares >= 192) return launch_product<E, KIND, Large>(p, stream);
  if (tiles(p.m, cols, 256, 128) * shares >= 160) return launch_product<E, KIND, Tall>(p, stream);
  if (tiles(p.m, cols, 128, 128) * shares >= 160) return launch_product<E, KIND, Middle>(p, stream);
  return launch_product<E, KIND, Small>(p, stream);
}

template <typename E, int KIND> int launch_rows(const Args& p, hipStream_t stream);  // feed_forward_rows.h
constexpr int kFewRows = 64;

template <typename E> int product_of(Kind kind, const Args& p, hipStream_t stream) {
  if (p.m <= kFewRows) {
    if (kind == LINEAR) return launch_rows<E, LINEAR>(p, stream);
    if (kind == GATED) return launch_rows<E, GATED>(p, stream);
  }
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
