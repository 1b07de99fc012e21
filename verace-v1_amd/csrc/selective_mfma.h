// Matrix-core pieces of the chunked selective scan and its backward.
//
// All products run on 16 x 16 tiles with operands in one fragment layout: lane l holds index l % 16 of the
// outer dimension and, for g = l / 16, the eight contraction indexes k0 + 4g + 0..3 and k0 + 16 + 4g + 0..3
// of a block of 32.  A product's accumulator (lane: column l % 16, rows 4g + 0..3) is then already half a
// fragment of the products that contract over its rows.
//   E = __bf16: one v_mfma_f32_16x16x32_bf16 per block, fp32 sums.  Operands that are not 16-bit inputs are
//     rounded to bf16, or split into as many bf16 parts as the result needs.
//   E = float: eight v_mfma_f32_16x16x4f32 (exact products): fp32 and fp16 inputs (fp16 cannot hold the
//     decayed sums' range, and bf16 not its 11 bits).
#pragma once

#include "selective.h"
#include "vmi_lanes.h"
#include "vmi_mfma.h"

namespace vmi {
namespace sel {

template <typename E> struct Frag;
template <> struct Frag<__bf16> { bf16x8 v; };
template <> struct Frag<float> { f32x4 v[2]; };

__device__ __forceinline__ f32x4 mma(const Frag<__bf16>& a, const Frag<__bf16>& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(const Frag<float>& a, const Frag<float>& b, f32x4 c) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[h][i], b.v[h][i], c, 0, 0, 0);
  return c;
}

// A row-major tile of W columns in LDS.  The pitch and the shift of every other eight 16-bit rows put both
// the row reads (16 rows by 16 bytes) and the transposing reads (8 rows by 32 bytes) in distinct banks; fp32
// rows likewise (16 rows by 16 bytes, 4 rows by 64).
template <typename E, int W> struct Tile {
  static constexpr int PITCH = sizeof(E) == 2 ? W + 16 : W + 4;
  static constexpr int elems(int rows) { return rows * PITCH; }
  static __device__ __forceinline__ int at(int row) { return row * PITCH + (sizeof(E) == 2 ? (row & 8) : 0); }
};

template <typename E, int W>
__device__ __forceinline__ Frag<E> row_frag(const E* tile, int row0, int k0, int l16, int g) {
  const E* p = tile + Tile<E, W>::at(row0 + l16) + k0 + 4 * g;
  Frag<E> f;
  if constexpr (sizeof(E) == 2) {
    f.v = cat8<bf16x4, bf16x8>(*reinterpret_cast<const bf16x4*>(p), *reinterpret_cast<const bf16x4*>(p + 16));
  } else {
    f.v[0] = *reinterpret_cast<const f32x4*>(p);
    f.v[1] = *reinterpret_cast<const f32x4*>(p + 16);
  }
  return f;
}
// The fragment whose outer index is a column and whose contraction runs down the rows.
template <typename E, int W>
__device__ __forceinline__ Frag<E> col_frag(const E* tile, int k0, int col0, int l16, int g) {
  Frag<E> f;
  if constexpr (sizeof(E) == 2) {
    typedef short i16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    const E* p = tile + Tile<E, W>::at(k0 + 4 * g + (l16 >> 2)) + col0 + 4 * (l16 & 3);
    const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p));
    const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p + 16 * Tile<E, W>::PITCH));
    f.v = cat8<bf16x4, bf16x8>(__builtin_bit_cast(bf16x4, a), __builtin_bit_cast(bf16x4, b));
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) f.v[h][i] = tile[Tile<E, W>::at(k0 + 16 * h + 4 * g + i) + col0 + l16];
  }
  return f;
}

// Two accumulator tiles (contraction indexes k0 + 4g + r and k0 + 16 + 4g + r) as a fragment, rounded once.
template <typename E> __device__ __forceinline__ Frag<E> acc_frag(f32x4 a, f32x4 b) {
  Frag<E> f;
  if constexpr (sizeof(E) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f.v[i] = static_cast<__bf16>(a[i]), f.v[4 + i] = static_cast<__bf16>(b[i]);
  } else {
    f.v[0] = a, f.v[1] = b;
  }
  return f;
}

// The parts of eight fp32 values: three bf16 parts hold all 24 bits, fp32 is its own part.
template <typename E> struct Parts { static constexpr int N = sizeof(E) == 2 ? 3 : 1; };
template <typename E>
__device__ __forceinline__ void split(const f32x4 (&x)[2], Frag<E> (&f)[Parts<E>::N]) {
  if constexpr (sizeof(E) == 2) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float r = x[h][i];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const __bf16 q = static_cast<__bf16>(r);
          f[k].v[4 * h + i] = q;
          r -= static_cast<float>(q);
        }
      }
  } else {
    f[0].v[0] = x[0], f[0].v[1] = x[1];
  }
}
template <typename E> __device__ __forceinline__ f32x4 half(const Frag<E>& f, int h) {
  if constexpr (sizeof(E) == 2) {
    f32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = static_cast<float>(f.v[4 * h + i]);
    return r;
  } else {
    return f.v[h];
  }
}

// Orders LDS accesses only: global loads and stores stay in flight across it.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);  // vmcnt(63) expcnt(7) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A tile's rows on their way from global memory: NTH threads hold PER 16-byte pieces each, all of one column.
// VEC: whole aligned pieces; else element by element.
template <typename IO, typename E, int W, int ROWS, int NTH, bool VEC> struct Stage {
  static constexpr int EL = 16 / sizeof(IO);
  static constexpr int PR = W / EL;                       // pieces of a row
  static constexpr int PER = (ROWS * PR + NTH - 1) / NTH;
  static constexpr int STEP = NTH / PR;                   // rows between a thread's pieces
  static_assert(NTH % PR == 0, "");
  uint4 v[PER];
  const IO* src;   // this thread's piece of row 0
  int64_t stride;
  int row, left;   // first row, and columns from the piece's first on
  __device__ __forceinline__ void init(const IO* base, int64_t stride_, int cols) {
    const int c = threadIdx.x % PR * EL;
    row = threadIdx.x / PR, left = cols - c, stride = stride_;
    src = base + row * stride + c;
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ uint4 piece(const IO* p) const {
    if constexpr (VEC) {
      return *reinterpret_cast<const uint4*>(p);
    } else {
      struct alignas(16) V { IO e[EL]; };
      V q = __builtin_bit_cast(V, make_uint4(0, 0, 0, 0));
#pragma unroll
      for (int j = 0; j < EL; ++j)
        if (j < left) q.e[j] = p[j];
      return __builtin_bit_cast(uint4, q);
    }
  }
  // rows t0 .. t0 + ROWS - 1, zeros from row `end` on
  __device__ __forceinline__ void fetch(int t0, int end) {
    if (left <= 0) return;
    const IO* p = src + t0 * stride;
    if (t0 + ROWS <= end) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (PER * NTH == ROWS * PR || row + STEP * i < ROWS) v[i] = piece(p + STEP * i * stride);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        v[i] = row + STEP * i < ROWS && t0 + row + STEP * i < end ? piece(p + STEP * i * stride) : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void commit(E* tile) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (PER * NTH != ROWS * PR && row + STEP * i >= ROWS) continue;
      E* dst = tile + Tile<E, W>::at(row + STEP * i) + threadIdx.x % PR * EL;
      if constexpr (sizeof(IO) == sizeof(E)) {
        *reinterpret_cast<uint4*>(dst) = v[i];
      } else {  // fp16 -> fp32
        const f16x8 h = __builtin_bit_cast(f16x8, v[i]);
#pragma unroll
        for (int k = 0; k < 2; ++k)
          *reinterpret_cast<float4*>(dst + 4 * k) =
              make_float4(static_cast<float>(h[4 * k]), static_cast<float>(h[4 * k + 1]), static_cast<float>(h[4 * k + 2]),
                          static_cast<float>(h[4 * k + 3]));
      }
    }
  }
};

// Log decays from a chunk's start, as two floats: their differences keep the accuracy of a small exponent.
__device__ __forceinline__ float decay(float2 to, float2 from) { return __expf((to.x - from.x) + (to.y - from.y)); }

}  // namespace sel
}  // namespace vmi
