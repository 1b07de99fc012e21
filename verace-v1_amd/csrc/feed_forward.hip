// The C entries of the feed-forward operators, and the two small kernels beside their products: the sum of the shares of a
// weight's gradient and the sum of a gradient over its rows.
//
//   y = residual + act(x W^T + b)                              2 M N K operations
//   h = act(x Wg^T) lin(x Wu^T)                                4 M F K
// backward, from the inputs alone or from the sums before the activation that the forward kept:
//   dz = dy act'(x W^T + b), dx = dz W, dW = dz^T x, db = sum dz
//   [dg du] likewise, dx = dg Wg + du Wu, [dWg; dWu] = [dg du]^T x
// dz is rounded once to x's type, as the matrix cores take it; products are summed in fp32.
#include "feed_forward.h"

using namespace vmi;
using namespace vmi::prod;

namespace {

constexpr int NTH = 256;
constexpr int64_t kMaxRow = INT64_C(1) << 24;  // bytes between rows: 128 of them lie within the 31 bits of a load's offset

// out = the sum of `splits` partial results of n elements.
template <typename T>
__global__ __launch_bounds__(NTH) void join_kernel(const float* partial, T* out, int64_t n, int splits) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * NTH + threadIdx.x) * 4;
  if (i >= n) return;
  float s[4], t[4];
  const int rest = n - i < 4 ? static_cast<int>(n - i) : 4;
  partial += i;
  load_cols<float, 4>(partial, 0, rest, s);
  for (int k = 1; k < splits; ++k) {
    load_cols<float, 4>(partial + k * n, 0, rest, t);
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] += t[j];
  }
  store_cols<T, 4>(out + i, 0, rest, s);
}

// dz from the kept sums (PAIR: [dg du] from [g u]), a 16-byte piece of the result a thread, zeros from column n to the row's end.
template <typename T, bool PAIR>
__global__ __launch_bounds__(NTH) void dz_kernel(const float* z, const T* dy, int64_t lddy, T* dz, int n, int whole, int64_t count, Gate gate) {
  constexpr int W = 16 / sizeof(T);
  const int64_t e = static_cast<int64_t>(blockIdx.x) * NTH + threadIdx.x;
  if (e >= count) return;
  const int pieces = whole / W, c = static_cast<int>(e % pieces) * W;
  const int64_t m = e / pieces;
  float d[W], a[W], b[W];
  T* out = dz + m * (PAIR ? 2 : 1) * whole;
  auto run = [&](auto full) {
    constexpr bool FULL = decltype(full)::value;
    load_cols<T, W, FULL>(dy + m * lddy, c, n, d);
    const float* row = z + m * (PAIR ? 2 : 1) * n;
    kept_cols<W, FULL>(row, c, n, a);
    if constexpr (PAIR) kept_cols<W, FULL>(row + n, c, n, b);
  };
  if (c + W <= n) run(std::true_type{});
  else run(std::false_type{});
  if constexpr (PAIR) {
    gated_slopes<T, W>(a, b, d, gate);
  } else {
    slope_all<T, W>(a, gate.act);
#pragma unroll
    for (int j = 0; j < W; ++j) a[j] *= d[j];
  }
#pragma unroll
  for (int j = 0; j < W; ++j) {
    a[j] = c + j < n ? a[j] : 0.f;
    if constexpr (PAIR) b[j] = c + j < n ? b[j] : 0.f;
  }
  store_cols<T, W, true>(out, c, whole, a);
  if constexpr (PAIR) store_cols<T, W, true>(out + whole, c, whole, b);
}

// Column sums of [rows, n]: workgroup (b, s) those of 256 columns over the s-th share of the rows.  A thread adds 8 columns of
// every eighth row (16 or 32 bytes a load), the eight are added in LDS.  One share alone is the result (out).
template <typename T>
__global__ __launch_bounds__(NTH) void columns_kernel(const T* x, int64_t ld, int rows, int n, int share, float* partial, T* out) {
  __shared__ float part[8][256];
  const int c = (threadIdx.x & 31) * 8, c0 = blockIdx.x * 256 + c, r0 = threadIdx.x >> 5;
  const int64_t first = static_cast<int64_t>(blockIdx.y) * share, last = rows - first < share ? rows : first + share;
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, t[8];
  auto add = [&](auto full) {
#pragma unroll 4
    for (int64_t r = first + r0; r < last; r += 8) {
      load_cols<T, 8, decltype(full)::value>(x + r * ld, c0, n, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += t[j];
    }
  };
  if (c0 + 8 <= n) add(std::true_type{});
  else if (c0 < n) add(std::false_type{});
#pragma unroll
  for (int j = 0; j < 8; ++j) part[r0][c + j] = s[j];
  __syncthreads();
  float sum = 0.f;
#pragma unroll
  for (int r = 0; r < 8; ++r) sum += part[r][threadIdx.x];
  if (const int col = blockIdx.x * 256 + threadIdx.x; col < n) {
    if (out != nullptr) io<T>::store(out, col, sum);
    else partial[static_cast<int64_t>(blockIdx.y) * n + col] = sum;
  }
}
// 32 columns a workgroup, each share's eighth by 32 threads.
template <typename T>
__global__ __launch_bounds__(NTH) void columns_join_kernel(const float* partial, int shares, int n, T* out) {
  __shared__ float part[8][32];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), r = threadIdx.x >> 5;
  float s = 0.f;
  if (c < n)
    for (int k = r; k < shares; k += 8) s += partial[static_cast<int64_t>(k) * n + c];
  part[r][threadIdx.x & 31] = s;
  __syncthreads();
  if (r != 0 || c >= n) return;
  for (int k = 1; k < 8; ++k) s += part[k][threadIdx.x & 31];
  io<T>::store(out, c, s);
}

// Rows of `bytes` to rows of whole 16-byte pieces, zeros behind them: a piece a thread.  Several matrices a launch, one a
// blockIdx.y: an operator's operands come together (64 rows, K 250, N 251 in bf16, host time of a call: linear 18.7 us for 24.6 with a
// launch each, gated 19.3 for 31.4).
struct Pad {
  const char* src;
  int64_t ld;
  char* dst;
  int64_t rows, bytes;
  uint32_t pieces, n;  // a row's, and all of the launch's
};
struct Pads {
  Pad pad[3];
};
__global__ __launch_bounds__(NTH) void pad_kernel(Pads pads) {
  const Pad p = pads.pad[blockIdx.y];
  const uint32_t e = blockIdx.x * NTH + threadIdx.x;
  if (e >= p.n) return;
  const uint32_t row = e / p.pieces;
  const int64_t at = static_cast<int64_t>(e - row * p.pieces) * 16;
  const char* from = p.src + row * p.ld + at;
  uint4 v = make_uint4(0, 0, 0, 0);
  if (at + 16 <= p.bytes) {
    __builtin_memcpy(&v, from, 16);
  } else {
    unsigned char* b = reinterpret_cast<unsigned char*>(&v);
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (at + j < p.bytes) b[j] = from[j];
  }
  *reinterpret_cast<uint4*>(p.dst + static_cast<int64_t>(e) * 16) = v;
}
int pad_status(const Pad& p) {
  if (p.rows < 0 || p.bytes < 0 || p.ld < 0) return VMI_ERR_INVALID_ARG;
  if (p.rows == 0 || p.bytes == 0) return VMI_OK;
  if (p.src == nullptr || p.dst == nullptr || reinterpret_cast<uintptr_t>(p.dst) % 16 != 0) return VMI_ERR_INVALID_ARG;
  if (p.bytes > INT64_MAX - 15 || p.rows > INT64_MAX / 16 / ((p.bytes + 15) / 16)) return VMI_ERR_INVALID_ARG;
  return (p.bytes + 15) / 16 > UINT32_MAX / NTH ? VMI_ERR_UNSUPPORTED : VMI_OK;
}
// All matrices' rows, as many of each as a launch takes at a time.
int pad_all(Pads p, hipStream_t stream) {
  for (const Pad& m : p.pad)
    if (const int st = pad_status(m); st != VMI_OK) return st;
  for (;;) {
    uint32_t most = 0, count = 0;
    for (int i = 0; i < 3; ++i) {
      Pad& m = p.pad[i];
      m.pieces = static_cast<uint32_t>((m.bytes + 15) / 16);
      const int64_t per = m.pieces == 0 ? 0 : UINT32_MAX / NTH * NTH / m.pieces, rows = m.rows < per ? m.rows : per;
      m.n = static_cast<uint32_t>(rows * m.pieces);
      if (m.n > most) most = m.n;
      if (m.n > 0) count = i + 1;
    }
    if (most == 0) return VMI_OK;
    hipLaunchKernelGGL(pad_kernel, dim3((most - 1) / NTH + 1, count), dim3(NTH), 0, stream, p);
    if (const int st = hip_status(hipGetLastError()); st != VMI_OK) return st;
    for (Pad& m : p.pad) {
      if (m.n == 0) continue;
      const int64_t rows = m.n / m.pieces;
      m.src += rows * m.ld, m.dst += static_cast<int64_t>(m.n) * 16, m.rows -= rows;
    }
  }
}

int product(int dtype, Kind kind, const Args& p, hipStream_t stream) {
  switch (dtype) {
    case VMI_BF16: return product_bf16(kind, p, stream);
    case VMI_F16: return product_f16(kind, p, stream);
    case VMI_F32: return product_f32(kind, p, stream);
    case VMI_E4M3: return product_e4m3(kind, p, stream);
  }
  return VMI_ERR_INVALID_ARG;
}

int64_t size_of(int dtype) { return dtype == VMI_F32 ? 4 : dtype == VMI_E4M3 ? 1 : 2; }
int64_t whole(int64_t n, int dtype) {  // elements of the 16-byte pieces that hold n
  const int64_t e = 16 / size_of(dtype);
  return (n + e - 1) / e * e;
}
size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// A matrix whose rows the tiles load in 16-byte pieces: a tile's rows lie within 31 bits of its first.
int rows_status(const void* p, int64_t rows, int64_t cols, int64_t ld, int dtype) {
  if (rows == 0 || cols == 0) return VMI_OK;
  if (p == nullptr || ld < cols) return VMI_ERR_INVALID_ARG;
  const int64_t size = size_of(dtype);
  if (reinterpret_cast<uintptr_t>(p) % 16 != 0 || ld * size % 16 != 0 || ld < whole(cols, dtype)) return VMI_ERR_UNSUPPORTED;
  return ld * size >= kMaxRow ? VMI_ERR_UNSUPPORTED : VMI_OK;
}
bool sizes_ok(int64_t m, int64_t n, int64_t k) {
  const int64_t most = INT64_C(1) << 30;
  return m >= 0 && n >= 0 && k >= 0 && m <= most && n <= most && k <= most;
}
int first_error(std::initializer_list<int> status) {
  for (int s : status)
    if (s != VMI_OK) return s;
  return VMI_OK;
}

// Shares of dW's contraction: as many as fill the compute units once with tiles of 256 x 128, each of 512 rows at least.
struct Shares {
  int n, length;
};
Shares weight_shares(int64_t rows, int64_t cols, int64_t k) {
  const int64_t t = tiles(rows, cols, 256, 128);
  int64_t n = t == 0 ? 1 : 256 / t;
  const int64_t most = (k + 511) / 512;
  if (n > most) n = most;
  if (n < 1) n = 1;
  int64_t length = ((k + n - 1) / n + 127) / 128 * 128;
  if (length < 128) length = 128;
  n = (k + length - 1) / length;
  return {static_cast<int>(n < 1 ? 1 : n), static_cast<int>(length)};
}
// dW [segments * valid, cols] = dz^T x over m rows.
int weight_gradient(const void* dz, int64_t lddz, int segments, int64_t seg, int64_t valid, const void* x, int64_t ldx,
                    int dtype, int64_t m, int64_t cols, void* dw, float* partial, hipStream_t stream) {
  if (valid == 0 || cols == 0) return VMI_OK;
  const Shares s = weight_shares(segments * seg, cols, m);
  Args p{};
  p.a = dz, p.lda = lddz, p.b = x, p.ldb = ldx;
  p.m = static_cast<int>(segments * seg), p.n = static_cast<int>(cols), p.k = static_cast<int>(m);
  p.splits = s.n, p.split_k = s.length, p.seg = static_cast<int>(seg), p.seg_valid = static_cast<int>(valid);
  p.out = dw, p.ldo = cols, p.partial = s.n > 1 ? partial : nullptr;
  if (const int st = product(dtype, DW, p, stream); st != VMI_OK || s.n == 1) return st;
  const int64_t n = segments * valid * cols, blocks = (n + 4 * NTH - 1) / (4 * NTH);
  if (!grid_fits(blocks, NTH)) return VMI_ERR_UNSUPPORTED;
  return by_type(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    hipLaunchKernelGGL(join_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(NTH), 0, stream, partial, static_cast<T*>(dw), n,
                       s.n);
    return hip_status(hipGetLastError());
  });
}
size_t weight_bytes(int64_t rows, int64_t valid, int64_t cols, int64_t m) {
  const Shares s = weight_shares(rows, cols, m);
  return s.n > 1 ? align256(static_cast<size_t>(s.n) * valid * cols * 4) : 0;
}
// dz [m, whole] (pair: [m, 2 whole]) from the sums that the forward kept.
int dz_from_kept(int dtype, bool pair, const float* kept, const void* dy, int64_t lddy, void* dz, int64_t m, int64_t n, const Gate& gate,
                 hipStream_t stream) {
  const int64_t w = whole(n, dtype), per_row = w / (16 / size_of(dtype));
  const int64_t rows_most = UINT32_MAX / NTH / per_row * NTH;
  if (rows_most == 0) return VMI_ERR_UNSUPPORTED;
  return by_type(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    const int parts = pair ? 2 : 1;
    for (int64_t row = 0; row < m; row += rows_most) {
      const int64_t count = (m - row < rows_most ? m - row : rows_most) * per_row;
      const dim3 grid(static_cast<unsigned>((count + NTH - 1) / NTH));
      const float* z = kept + row * parts * n;
      const T* d = static_cast<const T*>(dy) + row * lddy;
      T* out = static_cast<T*>(dz) + row * parts * w;
      if (pair)
        hipLaunchKernelGGL((dz_kernel<T, true>), grid, dim3(NTH), 0, stream, z, d, lddy, out, static_cast<int>(n), static_cast<int>(w), count, gate);
      else
        hipLaunchKernelGGL((dz_kernel<T, false>), grid, dim3(NTH), 0, stream, z, d, lddy, out, static_cast<int>(n), static_cast<int>(w), count, gate);
      if (const int st = hip_status(hipGetLastError()); st != VMI_OK) return st;
    }
    return VMI_OK;
  });
}
int column_shares(int64_t m, int64_t n) {
  const int64_t t = (n + 255) / 256, want = t == 0 ? 1 : (256 + t - 1) / t, most = (m + 31) / 32;
  const int64_t s = m <= 128 ? 1 : want < most ? want : most;  // 128 rows are 16 loads a thread, less than a second launch
  return static_cast<int>(s < 1 ? 1 : s);
}
Gate gate_of(int act, float beta1, float beta2) { return {act, beta1, beta2, 1.f / beta1, 1.f / beta2}; }
// 2^-64 to 2^64: a beta and its inverse times any value of a projection of ordinary size stay in fp32's range.
bool beta_ok(float b) { return b >= 0x1p-64f && b <= 0x1p64f; }
bool gate_ok(int act, float beta1, float beta2) { return act == ACT_SILU || (act == ACT_SITU && beta_ok(beta1) && beta_ok(beta2)); }
bool linear_act(int act) { return act == ACT_NONE || act == ACT_SILU || act == ACT_GELU; }

}  // namespace

extern "C" int vmi_pad_rows(const void* src, int64_t ld_bytes, void* dst, int64_t rows, int64_t row_bytes, void* stream) {
  const Pads p = {{{static_cast<const char*>(src), ld_bytes, static_cast<char*>(dst), rows, row_bytes, 0, 0}}};
  return pad_all(p, static_cast<hipStream_t>(stream));
}

extern "C" int vmi_pad_rows_3(const void* src0, int64_t ld_bytes0, void* dst0, int64_t rows0, int64_t row_bytes0, const void* src1,
                              int64_t ld_bytes1, void* dst1, int64_t rows1, int64_t row_bytes1, const void* src2, int64_t ld_bytes2,
                              void* dst2, int64_t rows2, int64_t row_bytes2, void* stream) {
  const Pads p = {{{static_cast<const char*>(src0), ld_bytes0, static_cast<char*>(dst0), rows0, row_bytes0, 0, 0},
                   {static_cast<const char*>(src1), ld_bytes1, static_cast<char*>(dst1), rows1, row_bytes1, 0, 0},
                   {static_cast<const char*>(src2), ld_bytes2, static_cast<char*>(dst2), rows2, row_bytes2, 0, 0}}};
  return pad_all(p, static_cast<hipStream_t>(stream));
}

extern "C" int vmi_feed_forward_form(int product, int dtype, int act, int64_t M, int64_t N, int64_t K, int* form) {
  if (form == nullptr || !sizes_ok(M, N, K) || dtype < 0 || dtype > VMI_E4M3 || product < 0 || product > 7) return VMI_ERR_INVALID_ARG;
  const bool gated = (product & 1) != 0;
  if (gated ? act != ACT_SILU && act != ACT_SITU : !linear_act(act)) return VMI_ERR_INVALID_ARG;
  if (dtype == VMI_E4M3 && product > 1) return VMI_ERR_INVALID_ARG;
  Args p{};
  p.gate.act = act, p.splits = 1;
  int64_t m = M, n = N, k = K;
  Kind kind;
  switch (product / 2) {
    case 0: kind = gated ? GATED : LINEAR; break;
    case 1: kind = gated ? GATED_DZ : LINEAR_DZ; break;
    case 2: kind = DX, n = K, k = N; break;
    default:
      kind = DW, m = (gated ? 2 : 1) * whole(N, dtype), n = K, k = M;
      if (m > INT32_MAX) return VMI_ERR_UNSUPPORTED;
      p.splits = weight_shares(m, n, k).n;
  }
  p.m = static_cast<int>(m), p.n = static_cast<int>(n), p.k = static_cast<int>(k);
  *form = form_of(kind, static_cast<int>(size_of(dtype)), p);
  return VMI_OK;
}

extern "C" int vmi_linear_add(const void* x, int64_t ldx, const float* x_scale, const void* w, int64_t ldw, const float* w_scale,
                              int dtype, const void* bias, const void* residual, int64_t ldr, int act, void* out, int64_t ldo,
                              int out_dtype, float* keep, int64_t M, int64_t N, int64_t K, void* stream) {
  if (!sizes_ok(M, N, K) || !linear_act(act) || dtype < 0 || dtype > VMI_E4M3 || out_dtype < 0 || out_dtype > VMI_F16)
    return VMI_ERR_INVALID_ARG;
  if (dtype != VMI_E4M3 && out_dtype != dtype) return VMI_ERR_INVALID_ARG;
  if (M == 0 || N == 0) return VMI_OK;
  if (out == nullptr || ldo < N || (residual != nullptr && ldr < N) || (dtype == VMI_E4M3 && (x_scale == nullptr || w_scale == nullptr)))
    return VMI_ERR_INVALID_ARG;
  if (const int st = first_error({rows_status(x, M, K, ldx, dtype), rows_status(w, N, K, ldw, dtype)}); st != VMI_OK) return st;
  Args p{};
  p.a = x, p.lda = ldx, p.b = w, p.ldb = ldw, p.xs = x_scale, p.ws = w_scale;
  p.m = static_cast<int>(M), p.n = static_cast<int>(N), p.k = static_cast<int>(K);
  p.bias = bias, p.other = residual, p.ldother = ldr, p.act = act, p.out = out, p.ldo = ldo, p.out_dtype = out_dtype;
  p.keep = keep;
  return product(dtype, LINEAR, p, static_cast<hipStream_t>(stream));
}

extern "C" int vmi_gated_linear(const void* x, int64_t ldx, const float* x_scale, const void* w_gate, int64_t ldg,
                                const float* gate_scale, const void* w_up, int64_t ldu, const float* up_scale, int dtype, int act,
                                float beta1, float beta2, void* out, int64_t ldo, int out_dtype, float* keep, int64_t M, int64_t F,
                                int64_t K, void* stream) {
  if (!sizes_ok(M, F, K) || !gate_ok(act, beta1, beta2) || dtype < 0 || dtype > VMI_E4M3 || out_dtype < 0 || out_dtype > VMI_F16)
    return VMI_ERR_INVALID_ARG;
  if (dtype != VMI_E4M3 && out_dtype != dtype) return VMI_ERR_INVALID_ARG;
  if (M == 0 || F == 0) return VMI_OK;
  if (out == nullptr || ldo < F || (dtype == VMI_E4M3 && (x_scale == nullptr || gate_scale == nullptr || up_scale == nullptr)))
    return VMI_ERR_INVALID_ARG;
  if (ldg != ldu) return VMI_ERR_UNSUPPORTED;
  if (const int st = first_error({rows_status(x, M, K, ldx, dtype), rows_status(w_gate, F, K, ldg, dtype),
                                  rows_status(w_up, F, K, ldu, dtype)});
      st != VMI_OK)
    return st;
  Args p{};
  p.a = x, p.lda = ldx, p.b = w_gate, p.b2 = w_up, p.ldb = ldg, p.xs = x_scale, p.ws = gate_scale, p.ws2 = up_scale;
  p.m = static_cast<int>(M), p.n = static_cast<int>(F), p.k = static_cast<int>(K);
  p.gate = gate_of(act, beta1, beta2), p.out = out, p.ldo = ldo, p.out_dtype = out_dtype;
  p.keep = keep;
  return product(dtype, GATED, p, static_cast<hipStream_t>(stream));
}

extern "C" int vmi_linear_add_bwd_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype, int act, size_t* bytes) {
  if (bytes == nullptr || !sizes_ok(M, N, K) || !linear_act(act) || dtype < 0 || dtype > VMI_F16) return VMI_ERR_INVALID_ARG;
  const int64_t n = whole(N, dtype);
  size_t b = act == ACT_NONE ? 0 : align256(static_cast<size_t>(M) * n * size_of(dtype));
  b += weight_bytes(n, N, K, M);
  *bytes = b + align256(static_cast<size_t>(column_shares(M, N)) * N * 4);
  return VMI_OK;
}

extern "C" int vmi_linear_add_bwd(const void* x, int64_t ldx, const void* w, int64_t ldw, int dtype, const void* bias, int act,
                                  const float* kept, const void* dy, int64_t lddy, void* dx, void* dw, void* db, int64_t M, int64_t N, int64_t K,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  size_t need = 0;
  if (const int st = vmi_linear_add_bwd_workspace_bytes(M, N, K, dtype, act, &need); st != VMI_OK) return st;
  if (workspace_bytes < need || (need > 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)))
    return VMI_ERR_WORKSPACE;
  if (const int st = first_error({rows_status(x, M, K, ldx, dtype), rows_status(w, N, K, ldw, dtype), rows_status(dy, M, N, lddy, dtype)});
      st != VMI_OK)
    return st;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t size = size_of(dtype), n = whole(N, dtype);
  if (n * size >= kMaxRow) return VMI_ERR_UNSUPPORTED;  // dz
  char* at = static_cast<char*>(workspace);
  const void* dz = dy;
  int64_t lddz = lddy;
  if (act != ACT_NONE) {
    dz = at, lddz = n;
    at += align256(static_cast<size_t>(M) * n * size);
    if (M > 0 && N > 0 && kept != nullptr) {
      Gate gate{};
      gate.act = act;
      if (const int st = dz_from_kept(dtype, false, kept, dy, lddy, const_cast<void*>(dz), M, N, gate, s); st != VMI_OK) return st;
    } else if (M > 0 && N > 0) {
      Args p{};
      p.a = x, p.lda = ldx, p.b = w, p.ldb = ldw, p.m = static_cast<int>(M), p.n = static_cast<int>(N), p.k = static_cast<int>(K);
      p.bias = bias, p.other = dy, p.ldother = lddy, p.act = act, p.out = const_cast<void*>(dz), p.ldo = lddz;
      if (const int st = product(dtype, LINEAR_DZ, p, s); st != VMI_OK) return st;
    }
  }
  float* partial = reinterpret_cast<float*>(at);
  at += weight_bytes(n, N, K, M);
  if (dx != nullptr && M > 0 && K > 0) {
    Args p{};
    p.a = dz, p.lda = lddz, p.b = w, p.ldb = ldw, p.m = static_cast<int>(M), p.n = static_cast<int>(K), p.k = static_cast<int>(N);
    p.out = dx, p.ldo = K;
    if (const int st = product(dtype, DX, p, s); st != VMI_OK) return st;
  }
  if (dw != nullptr)
    if (const int st = weight_gradient(dz, lddz, 1, n, N, x, ldx, dtype, M, K, dw, partial, s); st != VMI_OK) return st;
  if (db != nullptr && N > 0) {
    const int shares = column_shares(M, N);
    const int share = static_cast<int>((M + shares - 1) / shares);
    float* sums = reinterpret_cast<float*>(at);
    return by_type(dtype, [&](auto tag) -> int {
      using T = decltype(tag);
      if (!grid_fits((N + 31) / 32, NTH)) return VMI_ERR_UNSUPPORTED;
      hipLaunchKernelGGL(columns_kernel<T>, dim3(static_cast<unsigned>((N + 255) / 256), static_cast<unsigned>(shares)), dim3(NTH), 0,
                         s, static_cast<const T*>(dz), lddz, static_cast<int>(M), static_cast<int>(N), share, sums,
                         shares == 1 ? static_cast<T*>(db) : nullptr);
      if (shares > 1)
        hipLaunchKernelGGL(columns_join_kernel<T>, dim3(static_cast<unsigned>((N + 31) / 32)), dim3(NTH), 0, s, sums, shares,
                         static_cast<int>(N), static_cast<T*>(db));
      return hip_status(hipGetLastError());
    });
  }
  return VMI_OK;
}

extern "C" int vmi_gated_linear_bwd_workspace_bytes(int64_t M, int64_t F, int64_t K, int dtype, size_t* bytes) {
  if (bytes == nullptr || !sizes_ok(M, F, K) || dtype < 0 || dtype > VMI_F16) return VMI_ERR_INVALID_ARG;
  const int64_t f = whole(F, dtype);
  *bytes = align256(static_cast<size_t>(M) * 2 * f * size_of(dtype)) + weight_bytes(2 * f, 2 * F, K, M);
  return VMI_OK;
}

extern "C" int vmi_gated_linear_bwd(const void* x, int64_t ldx, const void* w_gate, int64_t ldg, const void* w_up, int64_t ldu,
                                    int dtype, int act, float beta1, float beta2, const float* kept, const void* dh, int64_t lddh,
                                    void* dx, void* dw, int64_t M, int64_t F, int64_t K, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  size_t need = 0;
  if (const int st = vmi_gated_linear_bwd_workspace_bytes(M, F, K, dtype, &need); st != VMI_OK) return st;
  if (!gate_ok(act, beta1, beta2)) return VMI_ERR_INVALID_ARG;
  if (workspace_bytes < need || (need > 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)))
    return VMI_ERR_WORKSPACE;
  if (ldg != ldu) return VMI_ERR_UNSUPPORTED;
  if (const int st = first_error({rows_status(x, M, K, ldx, dtype), rows_status(w_gate, F, K, ldg, dtype),
                                  rows_status(w_up, F, K, ldu, dtype)});
      st != VMI_OK)
    return st;
  if (M > 0 && F > 0 && (dh == nullptr || lddh < F)) return VMI_ERR_INVALID_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t size = size_of(dtype), f = whole(F, dtype), lddz = 2 * f;
  if (lddz * size >= kMaxRow) return VMI_ERR_UNSUPPORTED;
  char* dz = static_cast<char*>(workspace);
  float* partial = reinterpret_cast<float*>(dz + align256(static_cast<size_t>(M) * lddz * size));
  if (M > 0 && F > 0 && kept != nullptr) {
    if (const int st = dz_from_kept(dtype, true, kept, dh, lddh, dz, M, F, gate_of(act, beta1, beta2), s); st != VMI_OK) return st;
  } else if (M > 0 && F > 0) {
    Args p{};
    p.a = x, p.lda = ldx, p.b = w_gate, p.b2 = w_up, p.ldb = ldg, p.m = static_cast<int>(M), p.n = static_cast<int>(F);
    p.k = static_cast<int>(K), p.other = dh, p.ldother = lddh, p.gate = gate_of(act, beta1, beta2);
    p.out = dz, p.ldo = lddz, p.second = f;
    if (const int st = product(dtype, GATED_DZ, p, s); st != VMI_OK) return st;
  }
  if (dx != nullptr && M > 0 && K > 0) {
    Args p{};
    p.a = dz, p.lda = lddz, p.b = w_gate, p.b2 = w_up, p.ldb = ldg, p.second = f;
    p.m = static_cast<int>(M), p.n = static_cast<int>(K), p.k = static_cast<int>(F);
    p.out = dx, p.ldo = K;
    if (const int st = product(dtype, DX, p, s); st != VMI_OK) return st;
  }
  if (dw != nullptr) return weight_gradient(dz, lddz, 2, f, F, x, ldx, dtype, M, K, dw, partial, s);
  return VMI_OK;
}
