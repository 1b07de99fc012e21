// 16-byte pieces of a row and the dispatch on an element type, shared by the element-wise kernels.
#pragma once

#include <initializer_list>

#include "vmi_common.h"

namespace vmi {

// 16 bytes of T
template <typename T> struct Vec {
  static constexpr int N = 16 / sizeof(T);
  T e[N];
};
template <typename T> __device__ __forceinline__ Vec<T> ldv(const T* p) {
  return __builtin_bit_cast(Vec<T>, *reinterpret_cast<const uint4*>(p));
}
template <typename T> __device__ __forceinline__ void stv(T* p, const Vec<T>& v) {
  *reinterpret_cast<uint4*>(p) = __builtin_bit_cast(uint4, v);
}
template <typename T> __device__ __forceinline__ T round_to(float x) {
  T r;
  io<T>::store(&r, 0, x);
  return r;
}
template <typename T> __device__ __forceinline__ float rounded(float x) {
  return io<T>::to_f32(round_to<T>(x));
}

// Elements i0 .. i0 + N - 1 of a row of d as fp32, zeros past its end: one 16-byte load where the rows
// are whole aligned pieces (vec), element loads otherwise.
template <typename T>
__device__ __forceinline__ void load_piece(const T* row, int i0, int d, bool vec, float (&x)[Vec<T>::N]) {
  constexpr int N = Vec<T>::N;
  if (vec) {
    const Vec<T> v = ldv(row + i0);
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = io<T>::to_f32(v.e[j]);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = i0 + j < d ? io<T>::load(row, i0 + j) : 0.f;
  }
}
// The compiler's own type of a memory type.
template <typename T> struct native { typedef T type; };
template <> struct native<bf16_t> { typedef __bf16 type; };
template <typename T>
__device__ __forceinline__ void store_piece(T* row, int i0, int d, bool vec, const float (&x)[Vec<T>::N]) {
  constexpr int N = Vec<T>::N;
  if (vec) {
    typename native<T>::type e[N];  // by the conversion instructions, two at a time
#pragma unroll
    for (int j = 0; j < N; ++j) e[j] = static_cast<typename native<T>::type>(x[j]);
    uint4 v;
    __builtin_memcpy(&v, e, 16);
    *reinterpret_cast<uint4*>(row + i0) = v;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (i0 + j < d) io<T>::store(row, i0 + j, x[j]);
  }
}

// How many of item b's T tokens count: its length within 0 .. T, or all.
__device__ __forceinline__ int length_of(const void* lengths, int lengths64, int T, int b) {
  if (lengths == nullptr) return T;
  const int64_t n = lengths64 ? static_cast<const int64_t*>(lengths)[b] : static_cast<const int32_t*>(lengths)[b];
  return static_cast<int>(n < 0 ? 0 : n > T ? T : n);
}

// sigmoid: the library's exp and a full division for an fp32 result, v_exp_f32 and v_rcp_f32 (a few
// 2^-24 relative) for a 16-bit one.
template <typename T> __device__ __forceinline__ float sigmoid_for(float x) {
  if constexpr (sizeof(T) == 4) return 1.f / (1.f + expf(-x));
  return __builtin_amdgcn_rcpf(1.f + __expf(-x));
}
template <typename F> inline int by_type(int dtype, F&& f) {
  if (dtype == VMI_F32) return f(float{});
  if (dtype == VMI_BF16) return f(bf16_t{});
  if (dtype == VMI_F16) return f(f16_t{});
  return VMI_ERR_INVALID_ARG;
}
// Whether a grid dimension holds this many workgroups of so many threads.  Its threads are counted in 32 bits: a larger
// launch is cut to what is left of their number, without an error.
inline bool grid_fits(int64_t workgroups, int threads) { return workgroups <= UINT32_MAX / threads; }
// f(first, count) over n units in runs that a grid holds, `per` of them a workgroup of so many threads.
template <typename F> inline int in_launches(int64_t n, int threads, int64_t per, F&& f) {
  const int64_t most = UINT32_MAX / threads * per;
  for (int64_t i = 0; i < n; i += most)
    if (const int st = f(i, n - i < most ? n - i : most); st != 0) return st;
  return 0;
}
// p, `elements` further on (null stays null).
template <typename T> inline T* advance(const void* p, int64_t elements) {
  return p == nullptr ? nullptr : static_cast<T*>(const_cast<void*>(p)) + elements;
}
inline bool aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  return true;
}

}  // namespace vmi
