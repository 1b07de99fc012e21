// The norms around a block with its gate and residual scale, forward and backward, a row each:
//
//   r = y i1 w1, i1 = 1 / sqrt(mean(y^2) + eps1)            the norm after the block (w1 absent: r = y)
//   s = residual + scale act(gate) r                         the residual stream
//   n = s i2 w2, i2 = 1 / sqrt(mean(s^2) + eps2)            the norm before the next block
//
// and, for u = dn w2, v = dr w1, dr = dt scale act(gate):
//   dt = ds + i2 (u - s i2^2 mean(u s))                      = dresidual
//   dy = i1 (v - y i1^2 mean(v y)),  dgate = dt scale r act'(gate)
//   dw1 = sum dr y i1,  dscale = sum dt act(gate) r,  dw2 = sum dn s i2        (over the rows)
//
// Everything between the loads and the stores is fp32; n is formed from s before s is rounded to its
// type, and the backward forms s again from the same inputs instead of reading the rounded one.
//
// Bound by memory: each input is read once and each output written once.  A row is held in registers by
// one wave (two 16-byte pieces a lane at most: rows of up to 1024 16-bit elements, no barrier), longer
// ones by a workgroup.  The weights' gradients are kept in registers over the rows that a workgroup takes
// and leave it as one partial row each; a second kernel adds the partials in a fixed order.  bf16 rows of 1024:
// forward 18.8 us at 84 MB (4.5 TB/s), 79 us and backward 164 us at 872 MB together (3.6 TB/s).  The 16-bit backward holds
// five inputs of a row and the next one's: three workgroups a compute unit leave 168 registers for rows of up to 2048
// elements, and 10 to 28 spill (unaligned rows 37 to 70); above 4096 about 95 (250).
#include <algorithm>
#include <type_traits>

#include "vmi_common.h"
#include "vmi_dispatch.h"
#include "vmi_lanes.h"
#include "vmi_vec.h"

namespace vmi {
namespace gnorm {

constexpr int NTH = 256;

struct Args {
  const void *y, *res, *gate, *w1, *scale, *w2;
  int64_t y_stride, r_stride, g_stride;  // elements between rows
  void *s, *n;
  float* stats;                          // [2][rows]: i1, i2 (or null)
  const void *ds, *dn;                   // backward: gradients of s and n, contiguous (or null)
  void *dy, *dres, *dgate;               // contiguous (or null)
  float* partial;                        // [blocks][3][d]: dw1, dscale, dw2 (or null)
  int64_t rows, row0;                    // row0: the launch's first
  int d, silu;
  float eps1, eps2;
  bool vec, wide;
};

// Sum over the G lanes of a row: a wave, two of a workgroup's four, or all (red: one float a wave; the barrier after
// the reads lets the next sum use it again).
template <int G> __device__ __forceinline__ float row_sum(float x, float* red) {
  x = half_pair_sum(row_pair_sum(row16_sum(x)));
  if constexpr (G > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[wave] = x;
    __syncthreads();
    x = G == 128 ? red[wave & ~1] + red[wave | 1] : (red[0] + red[1]) + (red[2] + red[3]);
    __syncthreads();
  }
  return x;
}

// N weights from element i on: whole 16-byte pieces where the rows are (wide), element loads otherwise.
template <typename W, int N> __device__ __forceinline__ void load_w(const void* base, int i, int d, bool wide, float (&x)[N]) {
  const W* p = static_cast<const W*>(base);
  constexpr int EL = Vec<W>::N;
  if (wide) {
#pragma unroll
    for (int q = 0; q < N / EL; ++q) {
      const Vec<W> v = ldv(p + i + q * EL);
#pragma unroll
      for (int j = 0; j < EL; ++j) x[q * EL + j] = io<W>::to_f32(v.e[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = i + j < d ? io<W>::load(p, i + j) : 0.f;
  }
}

// act(gate) and its derivative, from the gate and its sigmoid
__device__ __forceinline__ float activation(float g, float sg, bool silu) { return silu ? g * sg : sg; }
__device__ __forceinline__ float slope(float g, float sg, bool silu) {
  return silu ? sg * (1.f + g * (1.f - sg)) : sg * (1.f - sg);
}

template <typename T, typename W, int G, int NV>
__global__ __launch_bounds__(NTH) void forward_kernel(Args a) {
  constexpr int N = Vec<T>::N;
  __shared__ float red[NTH / 64];
  const int lane = threadIdx.x % G, d = a.d;
  const int64_t row = a.row0 + static_cast<int64_t>(blockIdx.x) * (NTH / G) + threadIdx.x / G;
  if (row >= a.rows) return;  // whole waves (G = 64) or never
  const T* y = static_cast<const T*>(a.y) + row * a.y_stride;
  const T* res = static_cast<const T*>(a.res) + row * a.r_stride;
  const T* gate = a.gate == nullptr ? nullptr : static_cast<const T*>(a.gate) + row * a.g_stride;
  float t[NV][N], x[NV][N], q[NV][N];
  float ss = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int i = (lane + G * v) * N;
    if (i >= d) break;
    load_piece(y, i, d, a.vec, t[v]);
    load_piece(res, i, d, a.vec, x[v]);
    if (gate != nullptr) load_piece(gate, i, d, a.vec, q[v]);
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if ((lane + G * v) * N >= d) break;
#pragma unroll
    for (int j = 0; j < N; ++j) ss = fmaf(t[v][j], t[v][j], ss);
  }
  float i1 = 1.f;
  if (a.w1 != nullptr) i1 = rsqrtf(row_sum<G>(ss, red) / d + a.eps1);
  ss = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int i = (lane + G * v) * N;
    if (i >= d) break;
    float w1[N], sc[N];
    if (a.w1 != nullptr) load_w<W>(a.w1, i, d, a.wide, w1);
    if (a.scale != nullptr) load_w<W>(a.scale, i, d, a.wide, sc);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float r = t[v][j] * i1;
      if (a.w1 != nullptr) r *= w1[j];
      if (gate != nullptr) r *= activation(q[v][j], sigmoid_for<T>(q[v][j]), a.silu);
      t[v][j] = a.scale != nullptr ? fmaf(sc[j], r, x[v][j]) : x[v][j] + r;
      ss = fmaf(t[v][j], t[v][j], ss);
    }
    store_piece(static_cast<T*>(a.s) + row * d, i, d, a.vec, t[v]);
  }
  if (a.stats != nullptr && lane == 0) a.stats[row] = i1;
  if (a.w2 == nullptr) return;
  const float i2 = rsqrtf(row_sum<G>(ss, red) / d + a.eps2);
  if (a.stats != nullptr && lane == 0) a.stats[a.rows + row] = i2;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int i = (lane + G * v) * N;
    if (i >= d) break;
    float w2[N];
    load_w<W>(a.w2, i, d, a.wide, w2);
#pragma unroll
    for (int j = 0; j < N; ++j) t[v][j] *= i2 * w2[j];
    store_piece(static_cast<T*>(a.n) + row * d, i, d, a.vec, t[v]);
  }
}

// N elements from i on as they lie in memory.
template <typename T, bool VEC> __device__ __forceinline__ Vec<T> raw(const T* row, int i, int d) {
  if constexpr (VEC) {
    return ldv(row + i);
  } else {
    Vec<T> v;
#pragma unroll
    for (int j = 0; j < Vec<T>::N; ++j) v.e[j] = i + j < d ? row[i + j] : round_to<T>(0.f);
    return v;
  }
}
template <typename T> __device__ __forceinline__ void widen(const Vec<T>& v, float (&x)[Vec<T>::N]) {
#pragma unroll
  for (int j = 0; j < Vec<T>::N; ++j) x[j] = io<T>::to_f32(v.e[j]);
}

template <bool VEC, int N> __device__ __forceinline__ void store_wide(float* row, int i, int d, const float (&x)[N]) {
  if constexpr (VEC) {
#pragma unroll
    for (int q = 0; q < N; q += 4) *reinterpret_cast<float4*>(row + i + q) = make_float4(x[q], x[q + 1], x[q + 2], x[q + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (i + j < d) row[i + j] = x[j];
  }
}

// A workgroup takes NTH / G rows at a time, the next ones' inputs on their way meanwhile.
// DG32: dgate is fp32.  (A template, not a branch: that one spills three more registers, 249 us for 242 at 32768 rows of
// 1024.)
template <typename T, typename W, int G, int NV, bool VEC, bool DG32>
__global__ __launch_bounds__(NTH, NV == 1 ? 3 : 1) void backward_kernel(Args a) {
  constexpr int N = Vec<T>::N, RW = NTH / G;
  __shared__ float red[NTH / 64];
  __shared__ float sums[RW > 1 ? 3 * G * NV * N : 1];
  const int lane = threadIdx.x % G, d = a.d;
  float b1[NV][N] = {}, bs[NV][N] = {}, b2[NV][N] = {};  // dw1, dscale, dw2
  const bool has_gate = a.gate != nullptr, has_s = a.ds != nullptr, has_n = a.dn != nullptr;
  Vec<T> ry[NV], rr[NV], rg[NV], rs[NV], rn[NV];
  float r1 = 1.f, r2 = 0.f;
  auto fetch = [&](int64_t row) {
    if (row >= a.rows) return;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = (lane + G * v) * N;
      if (i >= d) break;
      ry[v] = raw<T, VEC>(static_cast<const T*>(a.y) + row * a.y_stride, i, d);
      if (has_gate) rg[v] = raw<T, VEC>(static_cast<const T*>(a.gate) + row * a.g_stride, i, d);
      if (has_s) rs[v] = raw<T, VEC>(static_cast<const T*>(a.ds) + row * d, i, d);
      if (has_n) {
        rr[v] = raw<T, VEC>(static_cast<const T*>(a.res) + row * a.r_stride, i, d);
        rn[v] = raw<T, VEC>(static_cast<const T*>(a.dn) + row * d, i, d);
      }
    }
    if (a.w1 != nullptr) r1 = a.stats[row];
    if (has_n) r2 = a.stats[a.rows + row];
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * RW, mine = threadIdx.x / G;
  fetch(static_cast<int64_t>(blockIdx.x) * RW + mine);
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * RW; row0 < a.rows; row0 += step) {
    const int64_t row = row0 + mine;
    const bool on = row < a.rows;  // the others take part in the barriers
    const float i1 = r1, i2 = r2;
    float t[NV][N], yv[NV][N], q[NV][N], sg[NV][N], dt[NV][N], x[NV][N], z[NV][N];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      widen<T>(ry[v], yv[v]);
      widen<T>(rg[v], q[v]);
      widen<T>(rs[v], dt[v]);
      widen<T>(rr[v], x[v]);
      widen<T>(rn[v], z[v]);
      if (!has_s)
#pragma unroll
        for (int j = 0; j < N; ++j) dt[v][j] = 0.f;
    }
    fetch(row + step);
    float dot = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = (lane + G * v) * N;
      if (i >= d) break;
      if (!on) break;
      if (has_gate)
#pragma unroll
        for (int j = 0; j < N; ++j) sg[v][j] = sigmoid_for<T>(q[v][j]);
      if (!has_n) continue;
      float w1[N], sc[N], w2[N];
      if (a.w1 != nullptr) load_w<W>(a.w1, i, d, a.wide, w1);
      if (a.scale != nullptr) load_w<W>(a.scale, i, d, a.wide, sc);
      load_w<W>(a.w2, i, d, a.wide, w2);
#pragma unroll
      for (int j = 0; j < N; ++j) {  // s again, u = dn w2 and u . s
        float r = yv[v][j] * i1;
        if (a.w1 != nullptr) r *= w1[j];
        if (has_gate) r *= activation(q[v][j], sg[v][j], a.silu);
        const float s = a.scale != nullptr ? fmaf(sc[j], r, x[v][j]) : x[v][j] + r;
        b2[v][j] = fmaf(z[v][j], s * i2, b2[v][j]);
        const float u = z[v][j] * w2[j];
        dot = fmaf(u, s, dot);
        t[v][j] = s;
        dt[v][j] = fmaf(i2, u, dt[v][j]);
      }
    }
    if (has_n) {
      const float m = row_sum<G>(dot, red) / d * i2 * i2 * i2;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if ((lane + G * v) * N >= d) break;
#pragma unroll
        for (int j = 0; j < N; ++j) dt[v][j] = fmaf(-m, t[v][j], dt[v][j]);
      }
    }
    dot = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = (lane + G * v) * N;
      if (i >= d || !on) break;
      if (a.dres != nullptr) store_piece(static_cast<T*>(a.dres) + row * d, i, d, VEC, dt[v]);
      float w1s[N], scs[N];
      if (a.w1 != nullptr) load_w<W>(a.w1, i, d, a.wide, w1s);
      if (a.scale != nullptr) load_w<W>(a.scale, i, d, a.wide, scs);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float w1 = a.w1 != nullptr ? w1s[j] : 1.f, sc = a.scale != nullptr ? scs[j] : 1.f;
        const float yn = yv[v][j] * i1;
        float act = 1.f, da = 0.f;
        if (has_gate) act = activation(q[v][j], sg[v][j], a.silu), da = slope(q[v][j], sg[v][j], a.silu);
        const float dr = dt[v][j] * sc * act;
        q[v][j] = dt[v][j] * sc * (yn * w1) * da;  // dgate
        bs[v][j] = fmaf(dt[v][j] * act, yn * w1, bs[v][j]);
        b1[v][j] = fmaf(dr, yn, b1[v][j]);
        dt[v][j] = dr * w1;
        dot = fmaf(dt[v][j], yv[v][j], dot);
      }
      if (a.dgate != nullptr) {
        if constexpr (DG32) store_wide<VEC>(static_cast<float*>(a.dgate) + row * d, i, d, q[v]);
        else store_piece(static_cast<T*>(a.dgate) + row * d, i, d, VEC, q[v]);
      }
    }
    float m = 0.f;
    if (a.w1 != nullptr) m = row_sum<G>(dot, red) / d * i1 * i1 * i1;
    if (a.dy == nullptr || !on) continue;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = (lane + G * v) * N;
      if (i >= d) break;
#pragma unroll
      for (int j = 0; j < N; ++j) dt[v][j] = fmaf(-m, yv[v][j], i1 * dt[v][j]);
      store_piece(static_cast<T*>(a.dy) + row * d, i, d, VEC, dt[v]);
    }
  }
  if (a.partial == nullptr) return;
  float* out = a.partial + static_cast<int64_t>(blockIdx.x) * 3 * d;
  if constexpr (RW > 1) {  // the rows' sums one after the other: the same order in every run
    constexpr int M = G * NV * N;
    for (int w = 0; w < RW; ++w) {
      if (mine == w) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const int i = (lane + G * v) * N + j;
            sums[i] = (w ? sums[i] : 0.f) + b1[v][j];
            sums[M + i] = (w ? sums[M + i] : 0.f) + bs[v][j];
            sums[2 * M + i] = (w ? sums[2 * M + i] : 0.f) + b2[v][j];
          }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < d; i += NTH) {
      out[i] = sums[i];
      out[d + i] = sums[M + i];
      out[2 * d + i] = sums[2 * M + i];
    }
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int i = (lane + G * v) * N + j;
        if (i >= d) continue;
        out[i] = b1[v][j];
        out[d + i] = bs[v][j];
        out[2 * d + i] = b2[v][j];
      }
  }
}

// dw[k][i] = sum of partial[b][k][i] over the blocks: 32 columns by 32 strided shares of the blocks.
template <typename W>
__global__ __launch_bounds__(1024) void weights_kernel(const float* __restrict__ partial, W* dw1, W* dscale, W* dw2,
                                                       int blocks, int d) {
  __shared__ float part[32][33];
  const int c = threadIdx.x & 31, share = threadIdx.x >> 5, col = blockIdx.x * 32 + c;
  float s = 0.f;
  if (col < 3 * d)
    for (int b = share; b < blocks; b += 32) s += partial[static_cast<int64_t>(b) * 3 * d + col];
  part[share][c] = s;
  __syncthreads();
  s = part[c][share];  // a column's shares in 32 neighbouring lanes
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor(s, off);
  const int out = blockIdx.x * 32 + share;
  if (c != 0 || out >= 3 * d) return;
  const int k = out / d, i = out - k * d;
  W* dst = k == 0 ? dw1 : k == 1 ? dscale : dw2;
  if (dst != nullptr) io<W>::store(dst, i, s);
}

// A wave takes rows of up to two pieces a lane, a workgroup longer ones; at most 8 pieces a lane.
template <typename T, bool BACKWARD, typename F> int by_row(int d, F&& f) {
  const int pieces = (d + Vec<T>::N - 1) / Vec<T>::N;
  if (pieces <= 64) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
  // two waves a row: one leaves 232 registers and no room for the next row's loads (220 us at 32768 rows of 1024)
  if (pieces <= 128) return f(std::integral_constant<int, BACKWARD ? 128 : 64>{}, std::integral_constant<int, BACKWARD ? 1 : 2>{});
  if (pieces <= 256) return f(std::integral_constant<int, NTH>{}, std::integral_constant<int, 1>{});
  if (pieces <= 512) return f(std::integral_constant<int, NTH>{}, std::integral_constant<int, 2>{});
  if (pieces <= 1024) return f(std::integral_constant<int, NTH>{}, std::integral_constant<int, 4>{});
  return VMI_ERR_UNSUPPORTED;
}
template <typename T, typename F> int by_weight(int w_dtype, int dtype, F&& f) {
  if (w_dtype == VMI_F32) return f(float{});
  if (w_dtype == dtype) return f(T{});
  return VMI_ERR_UNSUPPORTED;
}
bool rows_fit(int64_t d, int dtype) { return d <= (dtype == VMI_F32 ? 4096 : 8192); }

// Workgroups of the backward: enough to fill the card, and few enough that the partials stay small.
int backward_blocks(int64_t rows, int64_t d, int dtype) {
  const int64_t bytes = d * (dtype == VMI_F32 ? 4 : 2);
  const int per = bytes <= 1024 ? 4 : bytes <= 2048 ? 2 : 1;
  return static_cast<int>(std::min<int64_t>((rows + per - 1) / per, 768));
}

int check(const Args& a, int dtype, int w_dtype) {
  if (a.rows < 0 || a.d < 1 || a.silu < 0 || a.silu > 1) return VMI_ERR_INVALID_ARG;
  if (dtype < VMI_F32 || dtype > VMI_F16 || w_dtype < VMI_F32 || w_dtype > VMI_F16) return VMI_ERR_INVALID_ARG;
  if (a.rows > 0 && (a.y == nullptr || a.res == nullptr)) return VMI_ERR_INVALID_ARG;
  if (!rows_fit(a.d, dtype) || a.rows > INT32_MAX) return VMI_ERR_UNSUPPORTED;
  return VMI_OK;
}
bool vectors(const Args& a, int dtype) {
  const int n = dtype == VMI_F32 ? 4 : 8;
  return a.d % n == 0 && a.y_stride % n == 0 && a.r_stride % n == 0 && a.g_stride % n == 0 &&
         aligned16({a.y, a.res, a.gate, a.s, a.n, a.ds, a.dn, a.dy, a.dres, a.dgate});
}

}  // namespace gnorm
}  // namespace vmi

using namespace vmi;
using namespace vmi::gnorm;

extern "C" int vmi_gated_norm(const void* y, int64_t y_stride, const void* residual, int64_t r_stride,
                              const void* gate, int64_t g_stride, const void* w1, const void* scale,
                              const void* w2, int dtype, int w_dtype, int gate_act, float eps1, float eps2,
                              void* s, void* n, float* stats, int64_t rows, int64_t d, void* stream) {
  if (d < 1 || d > INT32_MAX) return VMI_ERR_INVALID_ARG;
  Args a{};
  a.y = y, a.res = residual, a.gate = gate, a.w1 = w1, a.scale = scale, a.w2 = w2;
  a.y_stride = y_stride, a.r_stride = r_stride, a.g_stride = gate == nullptr ? 0 : g_stride;
  a.s = s, a.n = n, a.stats = stats, a.rows = rows, a.d = static_cast<int>(d), a.silu = gate_act;
  a.eps1 = eps1, a.eps2 = eps2;
  if (const int st = check(a, dtype, w_dtype); st != VMI_OK) return st;
  if (rows == 0) return VMI_OK;
  if ((w2 != nullptr) != (n != nullptr) || s == nullptr) return VMI_ERR_INVALID_ARG;
  a.vec = vectors(a, dtype);
  a.wide = a.vec && aligned16({w1, scale, w2});
  return by_type(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    return by_weight<T>(w_dtype, dtype, [&](auto wtag) -> int {
      using W = decltype(wtag);
      return by_row<T, false>(a.d, [&](auto g, auto nv) -> int {
        constexpr int per = NTH / decltype(g)::value;
        return in_launches(rows, NTH, per, [&](int64_t row0, int64_t n) -> int {
          a.row0 = row0;
          hipLaunchKernelGGL((forward_kernel<T, W, decltype(g)::value, decltype(nv)::value>),
                             dim3(static_cast<unsigned>((n + per - 1) / per)), dim3(NTH), 0,
                             static_cast<hipStream_t>(stream), a);
          return hip_status(hipGetLastError());
        });
      });
    });
  });
}

extern "C" int vmi_gated_norm_bwd_workspace_bytes(int64_t rows, int64_t d, int dtype, size_t* bytes) {
  if (bytes == nullptr || rows < 0 || d < 1 || dtype < VMI_F32 || dtype > VMI_F16) return VMI_ERR_INVALID_ARG;
  if (!rows_fit(d, dtype) || rows > INT32_MAX) return VMI_ERR_UNSUPPORTED;
  *bytes = static_cast<size_t>(std::max(1, backward_blocks(rows, d, dtype))) * 3 * d * sizeof(float);
  return VMI_OK;
}

extern "C" int vmi_gated_norm_bwd(const void* y, int64_t y_stride, const void* residual, int64_t r_stride,
                                  const void* gate, int64_t g_stride, const void* w1, const void* scale,
                                  const void* w2, int dtype, int w_dtype, int gate_act, const float* stats,
                                  const void* ds, const void* dn, void* dy, void* dresidual, void* dgate,
                                  void* dw1, void* dscale, void* dw2, int64_t rows, int64_t d,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  if (d < 1 || d > INT32_MAX) return VMI_ERR_INVALID_ARG;
  Args a{};
  a.y = y, a.res = residual, a.gate = gate, a.w1 = w1, a.scale = scale, a.w2 = w2;
  a.y_stride = y_stride, a.r_stride = r_stride, a.g_stride = gate == nullptr ? 0 : g_stride;
  a.stats = const_cast<float*>(stats), a.ds = ds, a.dn = w2 == nullptr ? nullptr : dn;
  a.dy = dy, a.dres = dresidual, a.dgate = gate == nullptr ? nullptr : dgate;
  a.rows = rows, a.d = static_cast<int>(d), a.silu = gate_act & ~2;
  const bool dgate32 = gate_act & 2;
  if (const int st = check(a, dtype, w_dtype); st != VMI_OK) return st;
  if (rows > 0 && stats == nullptr && (w1 != nullptr || a.dn != nullptr)) return VMI_ERR_INVALID_ARG;
  const bool weights = dw1 != nullptr || dscale != nullptr || dw2 != nullptr;
  const int blocks = backward_blocks(rows, d, dtype);
  if (weights && rows > 0) {
    size_t need = 0;
    vmi_gated_norm_bwd_workspace_bytes(rows, d, dtype, &need);
    if (workspace == nullptr || workspace_bytes < need) return VMI_ERR_WORKSPACE;
    a.partial = static_cast<float*>(workspace);
  }
  if (rows == 0 && !weights) return VMI_OK;
  a.vec = vectors(a, dtype);
  a.wide = a.vec && aligned16({w1, scale, w2});
  hipStream_t st = static_cast<hipStream_t>(stream);
  return by_type(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    return by_weight<T>(w_dtype, dtype, [&](auto wtag) -> int {
      using W = decltype(wtag);
      int rc = VMI_OK;
      if (rows > 0)
        rc = by_row<T, true>(a.d, [&](auto g, auto nv) -> int {
          constexpr int G = decltype(g)::value, NV = decltype(nv)::value;
          const dim3 grid(static_cast<unsigned>(blocks));
          auto go = [&](auto vec, auto wide) -> int {
            hipLaunchKernelGGL((backward_kernel<T, W, G, NV, decltype(vec)::value, decltype(wide)::value>), grid, dim3(NTH), 0,
                               st, a);
            return hip_status(hipGetLastError());
          };
          if constexpr (sizeof(T) == 2)
            if (dgate32) return a.vec ? go(std::true_type{}, std::true_type{}) : go(std::false_type{}, std::true_type{});
          return a.vec ? go(std::true_type{}, std::false_type{}) : go(std::false_type{}, std::false_type{});
        });
      if (rc != VMI_OK || !weights) return rc;
      hipLaunchKernelGGL(weights_kernel<W>, dim3(static_cast<unsigned>((3 * d + 31) / 32)), dim3(1024), 0, st,
                         a.partial, static_cast<W*>(dw1), static_cast<W*>(dscale), static_cast<W*>(dw2), blocks,
                         a.d);
      return hip_status(hipGetLastError());
    });
  });
}
