// The feed-forward products for a few rows (a decode step): the weights are read straight into the matrix
// cores' operands, and a workgroup's eight waves take every eighth 128-byte step of the contraction of 16 columns (gated: 16
// of each projection).  Their sums are joined in LDS and finished by the same epilogue as the tiles'.  The rows of x come from
// the L2.  A wave has the loads of
// three or four steps in flight; what the epilogue reads is read ahead.  The latency of one access, the launch and, with many
// rows, x's bytes into each compute unit bound it.
#pragma once

#include "feed_forward.h"

namespace vmi {
namespace prod {

// An operand's bytes from `base` on, 2^31 at most; reads beyond, at kOutside, are zeros without a branch.
typedef __amdgpu_buffer_rsrc_t Bytes;
__device__ __forceinline__ Bytes bytes_from(const void* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, kOutside - 16, 0x20000);
}
// 16 rows of an operand over one step from element k0: lane l the 16-byte slots q and q + 4 of row l % 16, which starts at `row`.
template <typename E> __device__ __forceinline__ Frag load_rows(Bytes from, unsigned row, int k0, int k, int q) {
  constexpr int P = 16 / sizeof(E);
  const int lo = k0 + q * P, hi = lo + 4 * P;
  const unsigned at = row + lo * sizeof(E);
  Frag f;
  f.lo = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(from, lo < k ? at : kOutside, 0, 0));
  f.hi = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(from, hi < k ? at + 64 : kOutside, 0, 0));
  return f;
}

// MT: sixteens of rows.
template <typename E, int KIND, int MT> __global__ __launch_bounds__(512, 2) void rows_kernel(Args p) {
  constexpr bool PAIR = KIND == GATED;
  constexpr int KT = 128 / sizeof(E), WAVES = 8, B = PAIR ? 2 : 1;
  constexpr int AHEAD = B + MT <= 5 ? 4 : 3;  // steps whose loads are in flight: up to 160 registers
  __shared__ float part[WAVES][B][MT * 16][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
  // rows past the operand's end are its last
  const unsigned w_row = static_cast<unsigned>((n0 + i < p.n ? i : p.n - 1 - n0) * p.ldb * sizeof(E));
  Bytes w[B];
  w[0] = bytes_from(static_cast<const E*>(p.b) + n0 * p.ldb);
  if constexpr (PAIR) w[1] = bytes_from(static_cast<const E*>(p.b2) + n0 * p.ldb);
  const Bytes x = bytes_from(static_cast<const E*>(p.a) + m0 * p.lda);
  unsigned x_row[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
    x_row[t] = static_cast<unsigned>((m0 + t * 16 + i < p.m ? t * 16 + i : p.m - 1 - m0) * p.lda * sizeof(E));
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
      const int m = m0 + r0 + 32 * o;
      if (m >= p.m || r0 + 32 * o >= MT * 16) continue;
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
      for (int b = 0; b < B; ++b) fw[s][b] = load_rows<E>(w[b], w_row, k, p.k, q);
#pragma unroll
      for (int t = 0; t < MT; ++t) fx[s][t] = load_rows<E>(x, x_row[t], k, p.k, q);
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
      const int m = m0 + r0 + 32 * o;
      if (m >= p.m || r0 + 32 * o >= MT * 16 || n0 + c >= p.n) continue;
      float z[1] = {0.f}, z2[1] = {0.f};
#pragma unroll
      for (int v = 0; v < WAVES; ++v) {
        z[0] += part[v][0][r0 + 32 * o][c];
        if constexpr (PAIR) z2[0] += part[v][1][r0 + 32 * o][c];
      }
      finish<E, T, KIND, 1>(p, m, n0 + c, cols, z, z2, sizeof(E) == 1 ? xs[o] : 1.f, 0, other[o]);
    }
  });
}

template <typename E, int KIND, int MT> int launch_rows(const Args& p, hipStream_t stream) {
  const int64_t cols = (static_cast<int64_t>(p.n) + 15) / 16;
  if (!grid_fits(cols, 512)) return VMI_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(cols), static_cast<unsigned>((p.m + 16 * MT - 1) / (16 * MT)));
  hipLaunchKernelGGL((rows_kernel<E, KIND, MT>), grid, dim3(512), 0, stream, p);
  return hip_status(hipGetLastError());
}

}  // namespace prod
}  // namespace vmi
