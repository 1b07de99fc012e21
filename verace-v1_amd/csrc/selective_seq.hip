// Selective scan token by token: the single-token step in place, and short calls.
//
// Rows p of a head's state are independent: y[p] = sum_n S[p, n] C[n].  LPR lanes hold a row, four values
// each, and a wave takes 64 / LPR rows IT times over; the state stays in registers over the tokens.  The
// step is bound by the state's read and write (nontemporal, as every decode state here: it is touched once
// a token): at B64 H32 P64 N128 134 MB in 26.2 us, 5.1 TB/s.
#include <type_traits>

#include "selective.h"

namespace vmi {
namespace sel {

constexpr int NTH = 256;

template <typename T> __device__ __forceinline__ void load4(const T* p, int n0, int N, bool vec, float (&v)[4]) {
  if (vec && n0 < N) {
    struct alignas(4 * sizeof(T)) V4 { T e[4]; };
    const V4 q = *reinterpret_cast<const V4*>(p + n0);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = io<T>::to_f32(q.e[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = n0 + j < N ? io<T>::load(p, n0 + j) : 0.f;
  }
}

template <typename T, int LPR, int IT>
__global__ __launch_bounds__(NTH) void seq_kernel(Args a, int blocks_p, int64_t units, bool vec_state, bool vec_bc) {
  constexpr int RPI = 64 / LPR;
  const int lane = threadIdx.x & 63, n0 = 4 * (lane % LPR);
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (NTH / 64) + (threadIdx.x >> 6);
  if (unit >= units) return;
  const int64_t bh = unit / blocks_p;
  const int p0 = static_cast<int>(unit - bh * blocks_p) * (RPI * IT) + lane / LPR;
  const int b = static_cast<int>(bh / a.H), h = static_cast<int>(bh - static_cast<int64_t>(b) * a.H);
  const int g = h / (a.H / a.G);
  int n = length_of(a.lengths, a.lengths64, a.T, b);
  if (a.mask != nullptr && a.mask[b] == 0) n = 0;
  const bool in_place = a.state_in == a.state_out;
  float S[IT][4];
  if (n > 0 || !in_place) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int p = p0 + RPI * i;
      const int64_t o = (bh * a.P + p) * a.N + n0;
#pragma unroll
      for (int j = 0; j < 4; ++j) S[i][j] = 0.f;
      if (a.state_in == nullptr || p >= a.P) continue;
      if (vec_state && n0 < a.N) {
        const float4 v = ld_stream4(a.state_in + o);
        S[i][0] = v.x, S[i][1] = v.y, S[i][2] = v.z, S[i][3] = v.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n0 + j < a.N) S[i][j] = a.state_in[o + j];
      }
    }
  }
  const float A = a.A[h], D = a.D == nullptr ? 0.f : a.D[h], bias = a.bias == nullptr ? 0.f : a.bias[h];
  const T* x = static_cast<const T*>(a.x) + b * a.x_b + static_cast<int64_t>(h) * a.P;
  const T* bm = static_cast<const T*>(a.bm) + b * a.b_b + static_cast<int64_t>(g) * a.N;
  const T* cm = static_cast<const T*>(a.cm) + b * a.c_b + static_cast<int64_t>(g) * a.N;
  T* y = a.y == nullptr ? nullptr : static_cast<T*>(a.y) + (static_cast<int64_t>(b) * a.T * a.H + h) * a.P;
  const int64_t y_t = static_cast<int64_t>(a.H) * a.P;
  for (int t = 0; t < n; ++t) {
    const float d = step_size(load_scalar(a.delta, a.delta_dtype, b * a.d_b + t * a.d_t + h) + bias, a.softplus);
    const float decay = expf(d * A);
    float B[4], C[4], xv[IT], out[IT];
    load4(bm + t * a.b_t, n0, a.N, vec_bc, B);
    load4(cm + t * a.c_t, n0, a.N, vec_bc, C);
#pragma unroll
    for (int i = 0; i < IT; ++i) xv[i] = p0 + RPI * i < a.P ? io<T>::load(x + t * a.x_t, p0 + RPI * i) : 0.f;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const float dx = d * xv[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) S[i][j] = fmaf(decay, S[i][j], dx * B[j]);
      out[i] = (S[i][0] * C[0] + S[i][1] * C[1]) + (S[i][2] * C[2] + S[i][3] * C[3]);
    }
#pragma unroll
    for (int off = LPR / 2; off >= 1; off >>= 1)
#pragma unroll
      for (int i = 0; i < IT; ++i) out[i] += __shfl_xor(out[i], off);
    if (y != nullptr && n0 == 0)
#pragma unroll
      for (int i = 0; i < IT; ++i)
        if (p0 + RPI * i < a.P) io<T>::store(y + t * y_t, p0 + RPI * i, fmaf(D, xv[i], out[i]));
  }
  if (y != nullptr && n0 == 0)
    for (int t = n; t < a.T; ++t)
#pragma unroll
      for (int i = 0; i < IT; ++i)
        if (p0 + RPI * i < a.P) io<T>::store(y + t * y_t, p0 + RPI * i, 0.f);
  if (a.state_out == nullptr || (n == 0 && in_place)) return;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int p = p0 + RPI * i;
    if (p >= a.P) continue;
    const int64_t o = (bh * a.P + p) * a.N + n0;
    if (vec_state && n0 < a.N) {
      st_stream4(a.state_out + o, make_float4(S[i][0], S[i][1], S[i][2], S[i][3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + j < a.N) a.state_out[o + j] = S[i][j];
    }
  }
}

int launch_seq(const Args& a, int dtype, hipStream_t stream) {
  const int es = dtype == VMI_F32 ? 4 : 2;
  auto aligned = [&](const void* p, int64_t t, int64_t b) {
    return reinterpret_cast<uintptr_t>(p) % (4 * es) == 0 && t % 4 == 0 && b % 4 == 0;
  };
  const bool vec_state = a.N % 4 == 0 && aligned16({a.state_in, a.state_out});
  const bool vec_bc = a.N % 4 == 0 && aligned(a.bm, a.b_t, a.b_b) && aligned(a.cm, a.c_t, a.c_b);
  return by_type(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    auto go = [&](auto lpr, auto it) -> int {
      constexpr int rows = 64 / decltype(lpr)::value * decltype(it)::value;
      const int blocks_p = (a.P + rows - 1) / rows;
      const int64_t units = static_cast<int64_t>(a.B) * a.H * blocks_p, wgs = (units + NTH / 64 - 1) / (NTH / 64);
      if (!grid_fits(wgs, NTH)) return VMI_ERR_UNSUPPORTED;
      hipLaunchKernelGGL((seq_kernel<T, decltype(lpr)::value, decltype(it)::value>), dim3(static_cast<unsigned>(wgs)),
                         dim3(NTH), 0, stream, a, blocks_p, units, vec_state, vec_bc);
      return hip_status(hipGetLastError());
    };
    // eight rows' loads in flight a lane where that still leaves eight waves a compute unit, else two
    const bool many = static_cast<int64_t>(a.B) * a.H * a.P * a.N >= 2048LL * 2048;
    auto lanes = [&](auto lpr) -> int {
      return many ? go(lpr, std::integral_constant<int, 8>{}) : go(lpr, std::integral_constant<int, 2>{});
    };
    if (a.N <= 16) return lanes(std::integral_constant<int, 4>{});
    if (a.N <= 32) return lanes(std::integral_constant<int, 8>{});
    if (a.N <= 64) return lanes(std::integral_constant<int, 16>{});
    if (a.N <= 128) return lanes(std::integral_constant<int, 32>{});
    return lanes(std::integral_constant<int, 64>{});
  });
}

}  // namespace sel
}  // namespace vmi
