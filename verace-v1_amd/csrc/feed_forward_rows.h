// The feed-forward products for a few rows (a decode step, at most 64): the weights are read once, straight into the matrix
// cores' operands, and a workgroup's eight waves take every eighth 128-byte step of the contraction of 16 columns (gated: 16
// of each projection).  Their sums are joined in LDS and finished by the same epilogue as the tiles'.  The rows of x come from
// the L2.  A wave has the loads of
// three or four steps in flight; what the epilogue reads is read ahead.  The latency of one access, the launch and, with many
// rows, x's bytes into each compute unit bound it.
#pragma once

#include "feed_forward.h"

namespace vmi {
namespace prod {

// 16 rows of an operand over one step: lane l the 16-byte slots q and q + 4 of row l % 16, zeros past k.
template <typename E> __device__ __forceinline__ Frag load_rows(const E* row, int k0, int k, int q) {
  constexpr int P = 16 / sizeof(E);
  Frag f = {0, 0, 0, 0, 0, 0, 0, 0};
  const int lo = k0 + q * P, hi = lo + 4 * P;
  if (lo < k) f.lo = *reinterpret_cast<const i32x4*>(row + lo);
  if (hi < k) f.hi = *reinterpret_cast<const i32x4*>(row + hi);
  return f;
}

// MT: sixteens of rows.
template <typename E, int KIND, int MT> __global__ __launch_bounds__(512, 2) void rows_kernel(Args p) {
  constexpr bool PAIR = KIND == GATED;
  constexpr int KT = 128 / sizeof(E), WAVES = 8, B = PAIR ? 2 : 1;
  constexpr int AHEAD = B + MT <= 5 ? 4 : 3;  // steps whose loads are in flight: up to 160 registers
  __shared__ float part[WAVES][B][MT * 16][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16, n = n0 + i < p.n ? n0 + i : p.n - 1;
  const E* w[B];
  w[0] = static_cast<const E*>(p.b) + n * p.ldb;
  if constexpr (PAIR) w[1] = static_cast<const E*>(p.b2) + n * p.ldb;
  const E* x[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) x[t] = static_cast<const E*>(p.a) + (t * 16 + i < p.m ? t * 16 + i : p.m - 1) * p.lda;
  f32x4 acc[B][MT];
#pragma unroll
  for (int b = 0; b < B; ++b)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[b][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  // what the epilogue reads, ahead of the loop: this thread's results are row threadIdx / 16 + 32 o, column threadIdx % 16
  constexpr int OUT = (MT + 1) / 2;
  Columns<1> cols = {};
  float xs[OUT], other[OUT][1];
  const int c = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  auto read_ahead = [&](auto tag) {
    using T = decltype(tag);
    if (n0 + c >= p.n) return;
    cols = columns_at<E, T, KIND, 1>(p, n0 + c);
#pragma unroll
    for (int o = 0; o < OUT; ++o) {
      const int m = r0 + 32 * o;
      if (m >= p.m || m >= MT * 16) continue;
      if constexpr (sizeof(E) == 1) xs[o] = p.xs[m];
      if (KIND == LINEAR && p.other != nullptr) load_cols<T, 1>(static_cast<const T*>(p.other) + m * p.ldother, n0 + c, p.n, other[o]);
    }
  };
  by_result<E>(p, read_ahead);
  for (int k0 = wave * KT; k0 < p.k; k0 += AHEAD * WAVES * KT) {
    Frag fw[AHEAD][B], fx[AHEAD][MT];
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
      const int k = k0 + s * WAVES * KT;
#pragma unroll
      for (int b = 0; b < B; ++b) fw[s][b] = load_rows(w[b], k, p.k, q);
#pragma unroll
      for (int t = 0; t < MT; ++t) fx[s][t] = load_rows(x[t], k, p.k, q);
    }
#pragma unroll
    for (int s = 0; s < AHEAD; ++s)
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int b = 0; b < B; ++b) acc[b][t] = mma<E>(fw[s][b], fx[s][t], acc[b][t]);
  }
  // lane: columns 4 q .. of row i
#pragma unroll
  for (int b = 0; b < B; ++b)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) part[wave][b][t * 16 + i][4 * q + r] = acc[b][t][r];
  __syncthreads();
  by_result<E>(p, [&](auto tag) {
    using T = decltype(tag);
#pragma unroll
    for (int o = 0; o < OUT; ++o) {
      const int m = r0 + 32 * o;
      if (m >= p.m || m >= MT * 16 || n0 + c >= p.n) continue;
      float z[1] = {0.f}, z2[1] = {0.f};
#pragma unroll
      for (int v = 0; v < WAVES; ++v) {
        z[0] += part[v][0][m][c];
        if constexpr (PAIR) z2[0] += part[v][1][m][c];
      }
      finish<E, T, KIND, 1>(p, m, n0 + c, cols, z, z2, sizeof(E) == 1 ? xs[o] : 1.f, 0, other[o]);
    }
  });
}

template <typename E, int KIND> int launch_rows(const Args& p, hipStream_t stream) {
  const int64_t blocks = (static_cast<int64_t>(p.n) + 15) / 16;
  if (!grid_fits(blocks, 512)) return VMI_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (p.m <= 16) hipLaunchKernelGGL((rows_kernel<E, KIND, 1>), grid, dim3(512), 0, stream, p);
  else if (p.m <= 32) hipLaunchKernelGGL((rows_kernel<E, KIND, 2>), grid, dim3(512), 0, stream, p);
  else hipLaunchKernelGGL((rows_kernel<E, KIND, 4>), grid, dim3(512), 0, stream, p);
  return hip_status(hipGetLastError());
}

}  // namespace prod
}  // namespace vmi
