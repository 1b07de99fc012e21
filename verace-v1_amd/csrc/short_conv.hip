// Short causal depthwise convolution of a state space layer, forward, backward and single token:
//
//   z[t, c] = bias[c] + sum_j w[c, j] row[t - (K - 1) + j, c],   y = act(z),   K = 2 .. 4
//
// with row[t] = x[t] for t >= 0 and the K - 1 rows before them from the state [K - 1, C] (zeros without
// one); the state after n tokens is rows n - (K - 1) .. n - 1.  Of a sequence's T rows the first n (its
// length) are convolved; the others are neither read nor part of the state, and their y (and dx) are 0.
//
//   dz = dy act'(z);  drow[t] = sum_j w[j] dz[t + (K - 1) - j] (+ the state's gradient for its rows);
//   dw[j] = sum_t dz[t] row[t - (K - 1) + j],  dbias = sum_t dz[t]
//
// Bound by memory: x (and dy) read once, y (dx) written once; sums are fp32.  A thread takes four
// channels and slides down RUN tokens with the last K rows in registers, so the rows that
// two runs share (K - 1 of RUN) are the only ones read twice.  The weights' gradients leave a workgroup
// as one partial row per channel and are added by a second kernel in a fixed order.  B8 T4096 C2304 bf16: 65 us,
// 4.6 TB/s; backward at B4 T2048 C2304 fp32 65 us, 3.5 TB/s.
#include <algorithm>
#include <type_traits>

#include "vmi_common.h"
#include "vmi_dispatch.h"
#include "vmi_vec.h"

namespace vmi {
namespace sconv {

constexpr int NTH = 256;
constexpr int PIECE = 4;     // channels of a thread (one, where C or an address does not divide)
constexpr int RUN = 16;       // tokens of a thread, forward
constexpr int BRUN = 32;      // rows of a thread, backward
constexpr int CT = 64;        // channel pieces of a backward workgroup, by NTH / CT runs

struct Args {
  const void *x, *w, *bias, *state_in;
  void *y, *state_out;
  const void* lengths;         // [B] int32 or int64, or null
  const void *dy, *dstate_out;
  void *dx, *dstate_in;
  float* partial;              // [parts][C][K + 1]
  const uint8_t* mask;         // step: [B] or null
  int64_t x_stride, x_batch;   // elements between x's rows and items
  int64_t dy_stride, dy_batch;
  int B, T, C, w_dtype, act, lengths64;
  int pieces, runs;
  bool wide;                   // w and bias 16-byte aligned
};

// N consecutive elements as they lie in memory, N = 4 or 1.
template <typename T, int N> struct alignas(N * sizeof(T)) Raw { T e[N]; };
template <typename T, int N> __device__ __forceinline__ Raw<T, N> raw(const T* p) {
  return *reinterpret_cast<const Raw<T, N>*>(p);
}
template <typename T, int N> __device__ __forceinline__ void widen(const Raw<T, N>& r, float (&x)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) x[j] = io<T>::to_f32(r.e[j]);
}
template <typename T, int N> __device__ __forceinline__ void load(const T* p, float (&x)[N]) { widen<T, N>(raw<T, N>(p), x); }
template <typename T, int N> __device__ __forceinline__ void store(T* p, const float (&x)[N]) {
  Raw<T, N> r;
#pragma unroll
  for (int j = 0; j < N; ++j) r.e[j] = round_to<T>(x[j]);
  *reinterpret_cast<Raw<T, N>*>(p) = r;
}
template <int N> __device__ __forceinline__ void zero(float (&x)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) x[j] = 0.f;
}

// M consecutive parameters of type W from element i on, four at a time where wide.
template <typename W, int M>
__device__ __forceinline__ void parameters(const void* base, int64_t i, bool wide, float (&x)[M]) {
  const W* p = static_cast<const W*>(base) + i;
  if (M % 4 == 0 && wide) {
#pragma unroll
    for (int q = 0; q < M; q += 4) {
      const Raw<W, 4> v = raw<W, 4>(p + q);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[q + j] = io<W>::to_f32(v.e[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < M; ++j) x[j] = io<W>::load(p, j);
  }
}
template <int M>
__device__ __forceinline__ void parameters(const void* base, int dtype, int64_t i, bool wide, float (&x)[M]) {
  if (dtype == VMI_F32) parameters<float, M>(base, i, wide, x);
  else if (dtype == VMI_BF16) parameters<bf16_t, M>(base, i, wide, x);
  else parameters<f16_t, M>(base, i, wide, x);
}
// Weights and bias of channels c0 .. c0 + N - 1
template <typename T, int K, int N>
__device__ __forceinline__ void weights(const Args& a, int c0, float (&w)[K][N], float (&b)[N]) {
  float flat[K * N];
  parameters<K * N>(a.w, a.w_dtype, static_cast<int64_t>(c0) * K, a.wide, flat);
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][j] = flat[j * K + k];
  if (a.bias != nullptr) parameters<N>(a.bias, a.w_dtype, c0, a.wide, b);
  else zero(b);
}

// Row t of item b: the sequence's for t >= 0, the state's for -(K - 1) <= t < 0, zeros before.
template <typename T, int K, int N>
__device__ __forceinline__ void row(const Args& a, int b, int t, int c0, float (&x)[N]) {
  if (t >= 0)
    load<T, N>(static_cast<const T*>(a.x) + b * a.x_batch + t * a.x_stride + c0, x);
  else if (a.state_in != nullptr && t >= -(K - 1))
    load<T, N>(static_cast<const T*>(a.state_in) + (static_cast<int64_t>(b) * (K - 1) + (t + K - 1)) * a.C + c0, x);
  else
    zero(x);
}

template <typename T, int K, int N>
__device__ __forceinline__ void conv(const float (&w)[K][N], const float (&b)[N], const float (&win)[K][N], float (&z)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    z[j] = b[j];
#pragma unroll
    for (int k = 0; k < K; ++k) z[j] = fmaf(w[k][j], win[k][j], z[j]);
  }
}

// Threads of run `runs` (one past the tokens') copy the final state.
template <typename T, int K, int N>
__global__ __launch_bounds__(NTH) void forward_kernel(Args a) {
  const int id = blockIdx.x * NTH + threadIdx.x, b = blockIdx.y;
  const int run = id / a.pieces, c0 = (id - run * a.pieces) * N;
  if (run > a.runs) return;
  const int n = length_of(a.lengths, a.lengths64, a.T, b);
  if (run == a.runs) {
    if (a.state_out == nullptr) return;
    float x[N];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      row<T, K, N>(a, b, n - (K - 1) + k, c0, x);
      store<T, N>(static_cast<T*>(a.state_out) + (static_cast<int64_t>(b) * (K - 1) + k) * a.C + c0, x);
    }
    return;
  }
  const int t0 = run * RUN, t1 = min(t0 + RUN, a.T);
  T* y = static_cast<T*>(a.y) + (static_cast<int64_t>(b) * a.T + t0) * a.C + c0;
  float w[K][N], bias[N], win[K][N];
  Raw<T, N> next[RUN];
  weights<T, K, N>(a, c0, w, bias);
#pragma unroll
  for (int k = 0; k < K - 1; ++k) {
    if (t0 < n) row<T, K, N>(a, b, t0 - (K - 1) + k, c0, win[k + 1]);
    else zero(win[k + 1]);
  }
  const T* xr = static_cast<const T*>(a.x) + b * a.x_batch + t0 * a.x_stride + c0;
#pragma unroll
  for (int i = 0; i < RUN; ++i)  // every load of the run in flight at once
    if (t0 + i < n) next[i] = raw<T, N>(xr + i * a.x_stride);
#pragma unroll
  for (int i = 0; i < RUN; ++i) {
    if (t0 + i >= t1) break;
    float z[N];
    if (t0 + i < n) {
#pragma unroll
      for (int k = 0; k < K - 1; ++k)
#pragma unroll
        for (int j = 0; j < N; ++j) win[k][j] = win[k + 1][j];
      widen<T, N>(next[i], win[K - 1]);
      conv<T, K, N>(w, bias, win, z);
      if (a.act)
#pragma unroll
        for (int j = 0; j < N; ++j) z[j] *= sigmoid_for<T>(z[j]);
    } else {
      zero(z);
    }
    store<T, N>(y + static_cast<int64_t>(i) * a.C, z);
  }
}

// One token of every item: the state moves up a row.
template <typename T, int K, int N>
__global__ __launch_bounds__(64) void step_kernel(Args a) {
  const int id = blockIdx.x * blockDim.x + threadIdx.x, b = blockIdx.y, c0 = id * N;
  if (id >= a.pieces) return;
  float w[K][N], bias[N], win[K][N], z[N];
  zero(z);
  if (a.mask == nullptr || a.mask[b] != 0) {
    T* st = static_cast<T*>(a.state_out) + static_cast<int64_t>(b) * (K - 1) * a.C + c0;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) load<T, N>(st + static_cast<int64_t>(k) * a.C, win[k]);
    load<T, N>(static_cast<const T*>(a.x) + b * a.x_batch + c0, win[K - 1]);
    weights<T, K, N>(a, c0, w, bias);
    conv<T, K, N>(w, bias, win, z);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) store<T, N>(st + static_cast<int64_t>(k) * a.C, win[k + 1]);
    if (a.act)
#pragma unroll
      for (int j = 0; j < N; ++j) z[j] *= sigmoid_for<T>(z[j]);
  }
  store<T, N>(static_cast<T*>(a.y) + static_cast<int64_t>(b) * a.C + c0, z);
}

// A run is rows t0 .. t0 + BRUN - 1 counted from -(K - 1), so that the state's rows are the first run's
// first.  The pass goes down u = t0 .. t0 + BRUN + K - 2: z and dz of token u need rows u - (K - 1) .. u,
// and row u - (K - 1) is done once dz of u is known.
template <typename T, int K, int N>
__global__ __launch_bounds__(NTH, 3) void backward_kernel(Args a) {
  constexpr int RW = NTH / CT;
  __shared__ float sums[RW][K + 1][CT * N];
  const int cols = (a.pieces + CT - 1) / CT, part = blockIdx.x / cols, block = blockIdx.x - part * cols;
  const int piece = block * CT + threadIdx.x % CT, worker = threadIdx.x / CT;
  const int b = part / a.runs, run = (part - b * a.runs) * RW + worker;
  const int c0 = piece * N;
  const bool on = piece < a.pieces;
  float dw[K][N] = {}, db[N] = {};
  const int t0 = run * BRUN - (K - 1), t1 = min(t0 + BRUN, a.T);  // rows of this run
  if (on && t0 < a.T) {
    const int n = length_of(a.lengths, a.lengths64, a.T, b);
    float w[K][N], bias[N], win[K][N], dz[K][N];
    weights<T, K, N>(a, c0, w, bias);
#pragma unroll
    for (int k = 0; k < K; ++k) zero(dz[k]);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      if (t0 - (K - 1) + k < n) row<T, K, N>(a, b, t0 - (K - 1) + k, c0, win[k + 1]);
      else zero(win[k + 1]);
    }
    constexpr int GRP = 4;  // tokens whose loads are in flight together
#pragma unroll 1
    for (int u0 = t0; u0 < t1 + K - 1; u0 += GRP) {
      Raw<T, N> xs[GRP], gs[GRP];
#pragma unroll
      for (int i = 0; i < GRP; ++i) {
        const int u = u0 + i;
        if (u < 0 || u >= n || u >= t1 + K - 1) continue;
        xs[i] = raw<T, N>(static_cast<const T*>(a.x) + b * a.x_batch + u * a.x_stride + c0);
        if (a.dy != nullptr) gs[i] = raw<T, N>(static_cast<const T*>(a.dy) + b * a.dy_batch + u * a.dy_stride + c0);
      }
#pragma unroll
      for (int i = 0; i < GRP; ++i) {
        const int u = u0 + i;
        if (u >= t1 + K - 1) break;
#pragma unroll
        for (int k = 0; k < K - 1; ++k)
#pragma unroll
          for (int j = 0; j < N; ++j) {
            win[k][j] = win[k + 1][j];
            dz[k][j] = dz[k + 1][j];
          }
        zero(dz[K - 1]);
        if (u < n) {
          if (u < 0) {
            row<T, K, N>(a, b, u, c0, win[K - 1]);
          } else {
            widen<T, N>(xs[i], win[K - 1]);
            if (a.dy != nullptr) {
              float z[N], g[N];
              widen<T, N>(gs[i], g);
              conv<T, K, N>(w, bias, win, z);
#pragma unroll
              for (int j = 0; j < N; ++j) {
                if (a.act) {
                  const float sg = sigmoid_for<T>(z[j]);
                  g[j] *= sg * (1.f + z[j] * (1.f - sg));
                }
                dz[K - 1][j] = g[j];
              }
              if (u < t1) {  // token u is this run's
#pragma unroll
                for (int j = 0; j < N; ++j) {
                  db[j] += dz[K - 1][j];
#pragma unroll
                  for (int k = 0; k < K; ++k) dw[k][j] = fmaf(dz[K - 1][j], win[k][j], dw[k][j]);
                }
              }
            }
          }
        }
        const int t = u - (K - 1);  // done: dz of t .. t + K - 1 are dz[0] .. dz[K - 1]
        if (t < t0) continue;
        float d[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
          d[j] = 0.f;
#pragma unroll
          for (int k = 0; k < K; ++k) d[j] = fmaf(w[k][j], dz[K - 1 - k][j], d[j]);
        }
        if (a.dstate_out != nullptr && t < n && t >= n - (K - 1)) {
          float g[N];
          load<T, N>(static_cast<const T*>(a.dstate_out) + (static_cast<int64_t>(b) * (K - 1) + (t - n + K - 1)) * a.C + c0, g);
#pragma unroll
          for (int j = 0; j < N; ++j) d[j] += g[j];
        }
        if (t >= 0) {
          if (t >= n) zero(d);  // whatever the weights are
          if (t < a.T && a.dx != nullptr) store<T, N>(static_cast<T*>(a.dx) + (static_cast<int64_t>(b) * a.T + t) * a.C + c0, d);
        } else if (a.dstate_in != nullptr) {
          store<T, N>(static_cast<T*>(a.dstate_in) + (static_cast<int64_t>(b) * (K - 1) + (t + K - 1)) * a.C + c0, d);
        }
      }
    }
  }
  if (a.partial == nullptr) return;
  const int col = threadIdx.x % CT * N;
#pragma unroll
  for (int j = 0; j < N; ++j) {
#pragma unroll
    for (int k = 0; k < K; ++k) sums[worker][k][col + j] = dw[k][j];
    sums[worker][K][col + j] = db[j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < (K + 1) * CT * N; i += NTH) {
    const int k = i / (CT * N), c = i - k * (CT * N), ch = block * CT * N + c;
    if (ch >= a.C) continue;
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < RW; ++r) s += sums[r][k][c];
    a.partial[(static_cast<int64_t>(part) * a.C + ch) * (K + 1) + k] = s;
  }
}

// dw [C][K], dbias [C]: the sum of the parts, 64 values by 4 strided shares of them.
template <typename W>
__global__ __launch_bounds__(NTH) void weights_kernel(const float* __restrict__ partial, W* dw, W* dbias, int parts,
                                                      int C, int K) {
  __shared__ float p4[4][64];
  const int64_t total = static_cast<int64_t>(C) * (K + 1), i = static_cast<int64_t>(blockIdx.x) * 64 + (threadIdx.x & 63);
  const int share = threadIdx.x >> 6, l = threadIdx.x & 63;
  float s = 0.f;
  if (i < total)
    for (int p = share; p < parts; p += 4) s += partial[p * total + i];
  p4[share][l] = s;
  __syncthreads();
  if (share != 0 || i >= total) return;
  s = (p4[0][l] + p4[1][l]) + (p4[2][l] + p4[3][l]);
  const int64_t c = i / (K + 1);
  const int k = static_cast<int>(i - c * (K + 1));
  if (k < K) {
    if (dw != nullptr) io<W>::store(dw, c * K + k, s);
  } else if (dbias != nullptr) {
    io<W>::store(dbias, c, s);
  }
}

template <typename T, typename F> int by_shape(const Args& a, int K, bool vec, F&& f) {
  auto width = [&](auto n) -> int {
    if (K == 2) return f(std::integral_constant<int, 2>{}, n);
    if (K == 3) return f(std::integral_constant<int, 3>{}, n);
    return f(std::integral_constant<int, 4>{}, n);
  };
  return vec ? width(std::integral_constant<int, PIECE>{}) : width(std::integral_constant<int, 1>{});
}
bool vectors(const Args& a, int dtype) {
  const size_t bytes = PIECE * (dtype == VMI_F32 ? 4 : 2);
  for (const void* p : {a.x, a.state_in, static_cast<const void*>(a.y), static_cast<const void*>(a.state_out), a.dy,
                        a.dstate_out, static_cast<const void*>(a.dx), static_cast<const void*>(a.dstate_in)})
    if (reinterpret_cast<uintptr_t>(p) % bytes != 0) return false;
  return a.C % PIECE == 0 && a.x_stride % PIECE == 0 && a.x_batch % PIECE == 0 && a.dy_stride % PIECE == 0 &&
         a.dy_batch % PIECE == 0;
}
int check(int64_t B, int64_t T, int64_t C, int64_t K, int dtype, int w_dtype, int act) {
  if (B < 0 || T < 0 || C < 1 || K < 1 || act < 0 || act > 1) return VMI_ERR_INVALID_ARG;
  if (dtype < VMI_F32 || dtype > VMI_F16 || w_dtype < VMI_F32 || w_dtype > VMI_F16) return VMI_ERR_INVALID_ARG;
  if (K < 2 || K > 4 || T > INT32_MAX - 4096 || B > 65535 || C > (1 << 24)) return VMI_ERR_UNSUPPORTED;
  return VMI_OK;
}
int64_t backward_parts(int64_t B, int64_t T, int64_t K) {
  const int64_t rows = BRUN * (NTH / CT);
  return B * ((T + K - 1 + rows - 1) / rows);
}

}  // namespace sconv
}  // namespace vmi

using namespace vmi;
using namespace vmi::sconv;

extern "C" int vmi_short_conv(const void* x, int64_t x_stride, int64_t x_batch, const void* w, const void* bias,
                              int dtype, int w_dtype, int act, const void* state_in, const void* lengths,
                              int lengths64, void* y, void* state_out, int64_t B, int64_t T, int64_t C,
                              int64_t K, void* stream) {
  if (const int st = check(B, T, C, K, dtype, w_dtype, act); st != VMI_OK) return st;
  if (B == 0) return VMI_OK;
  if (w == nullptr || (T > 0 && (x == nullptr || y == nullptr))) return VMI_ERR_INVALID_ARG;
  if (state_out != nullptr && state_out == state_in) return VMI_ERR_ALIAS;
  Args a{};
  a.x = x, a.w = w, a.bias = bias, a.state_in = state_in, a.lengths = lengths, a.lengths64 = lengths64;
  a.y = y, a.state_out = state_out, a.x_stride = x_stride, a.x_batch = x_batch;
  a.B = static_cast<int>(B), a.T = static_cast<int>(T), a.C = static_cast<int>(C), a.w_dtype = w_dtype, a.act = act;
  const bool vec = vectors(a, dtype);
  a.wide = aligned16({a.w, a.bias});
  return by_type(dtype, [&](auto tag) -> int {
    using IO = decltype(tag);
    a.pieces = vec ? a.C / PIECE : a.C;
    a.runs = (a.T + RUN - 1) / RUN;
    const int64_t blocks = (a.pieces * (a.runs + 1LL) + NTH - 1) / NTH;
    if (blocks > INT32_MAX / NTH) return VMI_ERR_UNSUPPORTED;  // an item's pieces are counted in 31 bits
    return by_shape<IO>(a, static_cast<int>(K), vec, [&](auto k, auto n) -> int {
      hipLaunchKernelGGL((forward_kernel<IO, decltype(k)::value, decltype(n)::value>),
                         dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(B)), dim3(NTH), 0, static_cast<hipStream_t>(stream), a);
      return hip_status(hipGetLastError());
    });
  });
}

extern "C" int vmi_short_conv_step(const void* x, int64_t x_batch, const void* w, const void* bias, int dtype,
                                   int w_dtype, int act, const uint8_t* mask, void* state, void* y, int64_t B,
                                   int64_t C, int64_t K, void* stream) {
  if (const int st = check(B, 1, C, K, dtype, w_dtype, act); st != VMI_OK) return st;
  if (B == 0) return VMI_OK;
  if (x == nullptr || w == nullptr || state == nullptr || y == nullptr) return VMI_ERR_INVALID_ARG;
  Args a{};
  a.x = x, a.w = w, a.bias = bias, a.mask = mask, a.state_out = state, a.y = y, a.x_batch = x_batch;
  a.B = static_cast<int>(B), a.T = 1, a.C = static_cast<int>(C), a.w_dtype = w_dtype, a.act = act;
  const bool vec = vectors(a, dtype);
  a.wide = aligned16({a.w, a.bias});
  return by_type(dtype, [&](auto tag) -> int {
    using IO = decltype(tag);
    a.pieces = vec ? a.C / PIECE : a.C;
    return by_shape<IO>(a, static_cast<int>(K), vec, [&](auto k, auto n) -> int {
      hipLaunchKernelGGL((step_kernel<IO, decltype(k)::value, decltype(n)::value>),
                         dim3(static_cast<unsigned>((a.pieces + 63) / 64), static_cast<unsigned>(B)), dim3(64), 0, static_cast<hipStream_t>(stream), a);
      return hip_status(hipGetLastError());
    });
  });
}

extern "C" int vmi_short_conv_bwd_workspace_bytes(int64_t B, int64_t T, int64_t C, int64_t K, size_t* bytes) {
  if (bytes == nullptr) return VMI_ERR_INVALID_ARG;
  if (const int st = check(B, T, C, K, VMI_F32, VMI_F32, 0); st != VMI_OK) return st;
  *bytes = static_cast<size_t>(backward_parts(B, T, K)) * C * (K + 1) * sizeof(float);
  return VMI_OK;
}

extern "C" int vmi_short_conv_bwd(const void* x, int64_t x_stride, int64_t x_batch, const void* w, const void* bias,
                                  int dtype, int w_dtype, int act, const void* state_in, const void* lengths,
                                  int lengths64, const void* dy, int64_t dy_stride, int64_t dy_batch,
                                  const void* dstate_out, void* dx, void* dw, void* dbias, void* dstate_in,
                                  int64_t B, int64_t T, int64_t C, int64_t K, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (const int st = check(B, T, C, K, dtype, w_dtype, act); st != VMI_OK) return st;
  if (w == nullptr || (B > 0 && T > 0 && x == nullptr)) return VMI_ERR_INVALID_ARG;
  Args a{};
  a.x = x, a.w = w, a.bias = bias, a.state_in = state_in, a.lengths = lengths, a.lengths64 = lengths64;
  a.dy = dy, a.dstate_out = dstate_out, a.dx = dx, a.dstate_in = dstate_in;
  a.x_stride = x_stride, a.x_batch = x_batch, a.dy_stride = dy == nullptr ? 0 : dy_stride;
  a.dy_batch = dy == nullptr ? 0 : dy_batch;
  a.B = static_cast<int>(B), a.T = static_cast<int>(T), a.C = static_cast<int>(C), a.w_dtype = w_dtype, a.act = act;
  const int64_t parts = backward_parts(B, T, K);
  if (parts > INT32_MAX) return VMI_ERR_UNSUPPORTED;
  const bool weights = dw != nullptr || dbias != nullptr;
  if (weights && B > 0) {
    size_t need = 0;
    vmi_short_conv_bwd_workspace_bytes(B, T, C, K, &need);
    if (workspace == nullptr || workspace_bytes < need) return VMI_ERR_WORKSPACE;
    a.partial = static_cast<float*>(workspace);
  }
  const bool vec = vectors(a, dtype);
  a.wide = aligned16({a.w, a.bias});
  hipStream_t s = static_cast<hipStream_t>(stream);
  int rc = VMI_OK;
  if (B > 0)
    rc = by_type(dtype, [&](auto tag) -> int {
      using IO = decltype(tag);
      a.pieces = vec ? a.C / PIECE : a.C;
      a.runs = static_cast<int>(parts / B);
      const int64_t blocks = parts * ((a.pieces + CT - 1) / CT);
      if (!grid_fits(blocks, NTH)) return VMI_ERR_UNSUPPORTED;  // 2^37 elements and more
      return by_shape<IO>(a, static_cast<int>(K), vec, [&](auto k, auto n) -> int {
        hipLaunchKernelGGL((backward_kernel<IO, decltype(k)::value, decltype(n)::value>),
                           dim3(static_cast<unsigned>(blocks)), dim3(NTH), 0, s, a);
        return hip_status(hipGetLastError());
      });
    });
  if (rc != VMI_OK || !weights) return rc;
  return by_type(w_dtype, [&](auto tag) -> int {
    using W = decltype(tag);
    hipLaunchKernelGGL(weights_kernel<W>, dim3(static_cast<unsigned>((C * (K + 1) + 63) / 64)), dim3(NTH), 0, s,
                       a.partial, static_cast<W*>(dw), static_cast<W*>(dbias), static_cast<int>(parts), a.C,
                       static_cast<int>(K));
    return hip_status(hipGetLastError());
  });
}
