// The selective state space scan's shared pieces.
//
//   d_t = act(delta_t + bias),  a_t = exp(d_t A),  S_t = a_t S_{t-1} + d_t x_t B_t^T,  y_t = S_t C_t + D x_t
//
// per sequence b and head h, S [P, N]; heads h of a group share B and C.
#pragma once

#include "vmi_common.h"
#include "vmi_dispatch.h"
#include "vmi_vec.h"

namespace vmi {
namespace sel {

struct Args {
  const void *x, *delta, *bm, *cm;          // rows [H, P], [H], [G, N], [G, N] of token t, item b
  int64_t x_t, x_b, d_t, d_b, b_t, b_b, c_t, c_b;  // elements between tokens and between items
  const float *A, *D, *bias;                // [H]; D, bias may be null
  const float* state_in;                    // [B, H, P, N] or null (zeros)
  float* state_out;                         // or null
  void* y;                                  // [B, T, H, P] contiguous, or null
  const void* lengths;                      // [B] int32 or int64, or null
  const uint8_t* mask;                      // step: [B] or null
  int lengths64, delta_dtype, softplus;
  int B, T, H, P, G, N;
};

// The step size: softplus(z) = max(z, 0) + log1p(exp(-|z|)) with the library's functions (a few per token
// and head), or z itself.
__device__ __forceinline__ float step_size(float z, int softplus) {
  if (!softplus) return z;
  const float m = z > 0.f ? z : z != z ? z : 0.f;
  return m + log1pf(expf(-fabsf(z)));
}

// Workspace pieces start at multiples of 16 bytes.
inline int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }

// selective_seq.hip: token by token, any sizes with N <= 256.
int launch_seq(const Args& a, int dtype, hipStream_t stream);

// selective_chunk.hip: in chunks on the matrix cores, given the workspace; from use_chunk() tokens on.
bool use_chunk(int64_t B, int64_t T, int64_t H, int64_t P, int64_t N, int dtype);
size_t chunk_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t P, int64_t N, int dtype);
int launch_chunk(const Args& a, int dtype, void* workspace, hipStream_t stream);

// Step sizes and log decays of every chunk of L (32 or 64) tokens: d, c [B H][nch L].
int launch_prep(const Args& a, int L, float* d, float2* c, int nch, hipStream_t stream);

// selective_bwd.hip
struct Grads {
  const void* dy;            // [B, T, H, P], rows [H, P] at strides y_t, y_b
  int64_t y_t, y_b;
  const float* dstate;       // gradient of the final state, or null
  void *dx, *ddelta, *db, *dc;
  float *dA, *dD, *dbias, *dstate_in;
};
size_t bwd_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t P, int64_t G, int64_t N, int dtype);
int launch_bwd(const Args& a, int dtype, const Grads& q, void* workspace, hipStream_t stream);

}  // namespace sel
}  // namespace vmi
