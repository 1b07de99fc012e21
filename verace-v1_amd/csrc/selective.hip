// C entry points of the selective state space scan (selective.h).
#include <algorithm>
#include <initializer_list>

#include "selective_mfma.h"

using namespace vmi;
using namespace vmi::sel;

namespace {

int check(int64_t B, int64_t T, int64_t H, int64_t P, int64_t G, int64_t N, int dtype, int delta_dtype) {
  if (B < 0 || T < 0 || H < 1 || P < 1 || G < 1 || N < 1 || H % G != 0) return VMI_ERR_INVALID_ARG;
  if (dtype < VMI_F32 || dtype > VMI_F16 || delta_dtype < VMI_F32 || delta_dtype > VMI_F16) return VMI_ERR_INVALID_ARG;
  if (N > 256 || P > 1024 || T > INT32_MAX - 4096 || B > 65535 || H > 65535 || B * H > 4194304) return VMI_ERR_UNSUPPORTED;
  return VMI_OK;
}

// The chunk kernels' lane offsets are 32 bits wide and count up.
bool strides_fit(std::initializer_list<int64_t> strides, int64_t H, int64_t P) {
  for (int64_t s : strides)
    if (s < 0 || s > kMaxStride) return false;
  return H * P <= kMaxStride;
}

}  // namespace

extern "C" int vmi_selective_scan_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t P, int64_t G, int64_t N,
                                                  int dtype, size_t* bytes) {
  if (bytes == nullptr) return VMI_ERR_INVALID_ARG;
  if (const int st = check(B, T, H, P, G, N, dtype, VMI_F32); st != VMI_OK) return st;
  *bytes = chunk_workspace_bytes(B, T, H, P, N, dtype);
  return VMI_OK;
}

extern "C" int vmi_selective_scan_fwd(const void* x, int64_t x_t, int64_t x_b, const void* delta, int64_t d_t,
                                      int64_t d_b, int delta_dtype, const float* A, const void* bm, int64_t b_t,
                                      int64_t b_b, const void* cm, int64_t c_t, int64_t c_b, const float* D,
                                      const float* delta_bias, int softplus, int dtype, const float* state_in,
                                      const void* lengths, int lengths64, void* y, float* state_out, int64_t B,
                                      int64_t T, int64_t H, int64_t P, int64_t G, int64_t N, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  if (const int st = check(B, T, H, P, G, N, dtype, delta_dtype); st != VMI_OK) return st;
  if (B == 0) return VMI_OK;
  if (A == nullptr || state_out == nullptr) return VMI_ERR_INVALID_ARG;
  if (T > 0 && (x == nullptr || delta == nullptr || bm == nullptr || cm == nullptr)) return VMI_ERR_INVALID_ARG;
  if (state_out == state_in) return VMI_ERR_ALIAS;
  Args a{};
  a.x = x, a.delta = delta, a.bm = bm, a.cm = cm, a.x_t = x_t, a.x_b = x_b, a.d_t = d_t, a.d_b = d_b;
  a.b_t = b_t, a.b_b = b_b, a.c_t = c_t, a.c_b = c_b, a.A = A, a.D = D, a.bias = delta_bias;
  a.state_in = state_in, a.state_out = state_out, a.y = y, a.lengths = lengths, a.lengths64 = lengths64;
  a.delta_dtype = delta_dtype, a.softplus = softplus;
  a.B = static_cast<int>(B), a.T = static_cast<int>(T), a.H = static_cast<int>(H), a.P = static_cast<int>(P);
  a.G = static_cast<int>(G), a.N = static_cast<int>(N);
  if (!use_chunk(B, T, H, P, N, dtype) || !strides_fit({x_t, b_t, c_t}, H, P))
    return launch_seq(a, dtype, static_cast<hipStream_t>(stream));
  if (workspace == nullptr || workspace_bytes < chunk_workspace_bytes(B, T, H, P, N, dtype)) return VMI_ERR_WORKSPACE;
  return launch_chunk(a, dtype, workspace, static_cast<hipStream_t>(stream));
}

extern "C" int vmi_selective_scan_bwd_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t P, int64_t G,
                                                      int64_t N, int dtype, size_t* bytes) {
  if (bytes == nullptr) return VMI_ERR_INVALID_ARG;
  if (const int st = check(B, T, H, P, G, N, dtype, VMI_F32); st != VMI_OK) return st;
  *bytes = bwd_workspace_bytes(std::max<int64_t>(B, 1), std::max<int64_t>(T, 1), H, P, G, N, dtype);
  return VMI_OK;
}

extern "C" int vmi_selective_scan_bwd(const void* x, int64_t x_t, int64_t x_b, const void* delta, int64_t d_t,
                                      int64_t d_b, int delta_dtype, const float* A, const void* bm, int64_t b_t,
                                      int64_t b_b, const void* cm, int64_t c_t, int64_t c_b, const float* D,
                                      const float* delta_bias, int softplus, int dtype, const float* state_in,
                                      const void* lengths, int lengths64, const void* dy, int64_t y_t, int64_t y_b,
                                      const float* dstate, void* dx, void* ddelta, float* dA, void* db, void* dc,
                                      float* dD, float* dbias, float* dstate_in, int64_t B, int64_t T, int64_t H,
                                      int64_t P, int64_t G, int64_t N, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  if (const int st = check(B, T, H, P, G, N, dtype, delta_dtype); st != VMI_OK) return st;
  if (B == 0 || T == 0) return VMI_ERR_INVALID_ARG;  // nothing to differentiate
  if (A == nullptr || x == nullptr || delta == nullptr || bm == nullptr || cm == nullptr || dy == nullptr)
    return VMI_ERR_INVALID_ARG;
  if (!strides_fit({x_t, b_t, c_t, y_t}, H, P)) return VMI_ERR_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < bwd_workspace_bytes(B, T, H, P, G, N, dtype)) return VMI_ERR_WORKSPACE;
  Args a{};
  a.x = x, a.delta = delta, a.bm = bm, a.cm = cm, a.x_t = x_t, a.x_b = x_b, a.d_t = d_t, a.d_b = d_b;
  a.b_t = b_t, a.b_b = b_b, a.c_t = c_t, a.c_b = c_b, a.A = A, a.D = D, a.bias = delta_bias;
  a.state_in = state_in, a.lengths = lengths, a.lengths64 = lengths64, a.delta_dtype = delta_dtype, a.softplus = softplus;
  a.B = static_cast<int>(B), a.T = static_cast<int>(T), a.H = static_cast<int>(H), a.P = static_cast<int>(P);
  a.G = static_cast<int>(G), a.N = static_cast<int>(N);
  Grads q{dy, y_t, y_b, dstate, dx, ddelta, db, dc, dA, dD, dbias, dstate_in};
  return launch_bwd(a, dtype, q, workspace, static_cast<hipStream_t>(stream));
}

extern "C" int vmi_selective_step(const void* x, int64_t x_b, const void* delta, int64_t d_b, int delta_dtype,
                                  const float* A, const void* bm, int64_t b_b, const void* cm, int64_t c_b,
                                  const float* D, const float* delta_bias, int softplus, int dtype,
                                  const uint8_t* mask, float* state, void* y, int64_t B, int64_t H, int64_t P,
                                  int64_t G, int64_t N, void* stream) {
  if (const int st = check(B, 1, H, P, G, N, dtype, delta_dtype); st != VMI_OK) return st;
  if (B == 0) return VMI_OK;
  if (x == nullptr || delta == nullptr || A == nullptr || bm == nullptr || cm == nullptr || state == nullptr ||
      y == nullptr)
    return VMI_ERR_INVALID_ARG;
  Args a{};
  a.x = x, a.delta = delta, a.bm = bm, a.cm = cm, a.x_b = x_b, a.d_b = d_b, a.b_b = b_b, a.c_b = c_b;
  a.A = A, a.D = D, a.bias = delta_bias, a.state_in = state, a.state_out = state, a.y = y, a.mask = mask;
  a.delta_dtype = delta_dtype, a.softplus = softplus;
  a.B = static_cast<int>(B), a.T = 1, a.H = static_cast<int>(H), a.P = static_cast<int>(P);
  a.G = static_cast<int>(G), a.N = static_cast<int>(N);
  return launch_seq(a, dtype, static_cast<hipStream_t>(stream));
}
