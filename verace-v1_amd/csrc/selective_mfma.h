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

#include <type_traits>

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
// A tile that is only read by rows: the eight values of a lane's fragment lie side by side (one 16-byte read),
// and the four lane groups read from quarters a multiple of the banks apart, so that a read's 16 distinct rows
// are in distinct banks whichever lanes are served together.
template <typename E, int W> struct RowTile {
  static constexpr int PITCH = sizeof(E) == 2 ? (W == 32 ? 24 : W / 4 + 8) : W + 4;
  static constexpr int elems(int rows) { return rows * PITCH * (sizeof(E) == 2 ? 4 : 1); }
  // where the four elements from column c on (c % 4 == 0) lie in row r of a tile of ROWS
  template <int ROWS> static __device__ __forceinline__ int at(int r, int c) {
    if constexpr (sizeof(E) == 2) return ((c >> 2) & 3) * (ROWS * PITCH) + r * PITCH + (c >> 5) * 8 + ((c >> 4) & 1) * 4;
    else return r * PITCH + c;
  }
};
template <typename E, int W, int ROWS>
__device__ __forceinline__ Frag<E> packed_frag(const E* tile, int row0, int k0, int l16, int g) {
  const E* p = tile + (row0 + l16) * RowTile<E, W>::PITCH + (sizeof(E) == 2 ? g * (ROWS * RowTile<E, W>::PITCH) + k0 / 4 : k0 + 4 * g);
  Frag<E> f;
  if constexpr (sizeof(E) == 2) {
    f.v = *reinterpret_cast<const bf16x8*>(p);
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

// The parts that eight fp32 values are multiplied in: ALL hold their 24 bits (three of bf16), TERM is what a term of a
// 16-bit result takes (two: off by 2^-16 of it).  fp32 is its own part.
template <typename E> struct Parts {
  static constexpr int ALL = sizeof(E) == 2 ? 3 : 1;
  static constexpr int TERM = sizeof(E) == 2 ? 2 : 1;
};
// ALONE: the values are rows of different results, so none may see another's NaN.
template <typename E, int M, bool ALONE = false>
__device__ __forceinline__ void split(const f32x4 (&x)[2], Frag<E> (&f)[M]) {
  if constexpr (sizeof(E) == 2) {
    typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    // v - (its bf16) is exact, in one v_dot2 with a pair and (-1, 0) or (0, -1); a pair with an infinity gives NaN for
    // both, and both belong to one row of the product
    uint32_t first = 0x0000bf80u, second = 0xbf800000u;
    asm volatile("" : "+s"(first), "+s"(second));  // not as inline constants, whose place in a pair is the encoding's
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = x[i / 4][i % 4];
#pragma unroll
    for (int k = 0; k < M; ++k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[k].v[i] = static_cast<__bf16>(r[i]);  // v_cvt_pk_bf16_f32 pairs
      if (k == M - 1) break;
      const u32x4 q = __builtin_bit_cast(u32x4, f[k].v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t both = q[i];
        if constexpr (ALONE) {
          r[2 * i] -= __uint_as_float(both << 16);
          r[2 * i + 1] -= __uint_as_float(both & 0xffff0000u);
          continue;
        }
        const bf16x2 pair = __builtin_bit_cast(bf16x2, both);
        r[2 * i] = __builtin_amdgcn_fdot2_f32_bf16(pair, __builtin_bit_cast(bf16x2, first), r[2 * i], false);
        r[2 * i + 1] = __builtin_amdgcn_fdot2_f32_bf16(pair, __builtin_bit_cast(bf16x2, second), r[2 * i + 1], false);
      }
    }
  } else {
    f[0].v[0] = x[0], f[0].v[1] = x[1];
  }
}
// Half a fragment (four values side by side) as it is, to an aligned place.
__device__ __forceinline__ void put_half(__bf16* o, const Frag<__bf16>& f, int h) {
  *reinterpret_cast<bf16x4*>(o) = h ? __builtin_shufflevector(f.v, f.v, 4, 5, 6, 7) : __builtin_shufflevector(f.v, f.v, 0, 1, 2, 3);
}
__device__ __forceinline__ void put_half(float* o, const Frag<float>& f, int h) { *reinterpret_cast<f32x4*>(o) = f.v[h]; }
template <typename E> __device__ __forceinline__ f32x4 half(const Frag<E>& f, int h) {
  if constexpr (sizeof(E) == 2) {
    typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 q = __builtin_bit_cast(u32x4, f.v);
    return f32x4{__uint_as_float(q[2 * h] << 16), __uint_as_float(q[2 * h] & 0xffff0000u),
                 __uint_as_float(q[2 * h + 1] << 16), __uint_as_float(q[2 * h + 1] & 0xffff0000u)};
  } else {
    return f.v[h];
  }
}

// The number of this wave in its workgroup, known to be the same in all lanes.
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// Orders LDS accesses only: global loads and stores stay in flight across it.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);  // vmcnt(63) expcnt(7) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Elements between the rows of an input at most: 64 rows of fp32 from a tile's first in 32 bits.
constexpr int64_t kMaxStride = 1 << 23;

// A tile's rows on their way from global memory: NTH threads hold PER 16-byte pieces each, all of one column.
// VEC: whole aligned pieces; else element by element.
template <typename IO, typename E, int W, int ROWS, int NTH, bool VEC> struct Stage {
  static constexpr int EL = 16 / sizeof(IO);
  static constexpr int PR = W / EL;                       // pieces of a row
  static constexpr int PER = (ROWS * PR + NTH - 1) / NTH;
  static constexpr int STEP = NTH / PR;                   // rows between a thread's pieces
  static_assert(NTH % PR == 0, "");
  uint4 v[PER];
  const IO* src;   // row 0, the same in all lanes
  int64_t stride;
  uint32_t off;    // this thread's piece from there (kMaxStride keeps it in 32 bits)
  int row, left;   // first row, and columns from the piece's first on
  __device__ __forceinline__ void init(const IO* base, int64_t stride_, int cols) {
    const int c = threadIdx.x % PR * EL;
    row = threadIdx.x / PR, left = cols - c, stride = stride_, src = base;
    off = static_cast<uint32_t>(row) * static_cast<uint32_t>(stride) + c;
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
    const IO* p = src + t0 * stride;  // a scalar base and a lane's offset to every load
    if (t0 + ROWS <= end) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (PER * NTH == ROWS * PR || row + STEP * i < ROWS) v[i] = piece(p + STEP * i * stride + off);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        v[i] = row + STEP * i < ROWS && t0 + row + STEP * i < end ? piece(p + STEP * i * stride + off) : make_uint4(0, 0, 0, 0);
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
        *reinterpret_cast<float4*>(dst) = wide(i, 0);
        *reinterpret_cast<float4*>(dst + 4) = wide(i, 1);
      }
    }
  }
  __device__ __forceinline__ void commit_rows(E* tile) const {
    const int c = threadIdx.x % PR * EL;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (PER * NTH != ROWS * PR && row + STEP * i >= ROWS) continue;
      const int r = row + STEP * i;
      if constexpr (sizeof(E) == 2) {
        *reinterpret_cast<uint2*>(tile + RowTile<E, W>::template at<ROWS>(r, c)) = make_uint2(v[i].x, v[i].y);
        *reinterpret_cast<uint2*>(tile + RowTile<E, W>::template at<ROWS>(r, c + 4)) = make_uint2(v[i].z, v[i].w);
      } else if constexpr (sizeof(IO) == 4) {
        *reinterpret_cast<uint4*>(tile + RowTile<E, W>::template at<ROWS>(r, c)) = v[i];
      } else {
        *reinterpret_cast<float4*>(tile + RowTile<E, W>::template at<ROWS>(r, c)) = wide(i, 0);
        *reinterpret_cast<float4*>(tile + RowTile<E, W>::template at<ROWS>(r, c + 4)) = wide(i, 1);
      }
    }
  }
  __device__ __forceinline__ float4 wide(int i, int h) const {
    const f16x8 q = __builtin_bit_cast(f16x8, v[i]);
    return make_float4(static_cast<float>(q[4 * h]), static_cast<float>(q[4 * h + 1]), static_cast<float>(q[4 * h + 2]),
                       static_cast<float>(q[4 * h + 3]));
  }
};

// fp32 -> four values of the memory type, by the conversion instructions.
template <typename IO> struct alignas(4 * sizeof(IO)) Out4 { IO e[4]; };
template <typename IO> __device__ __forceinline__ Out4<IO> out4(f32x4 x) {
  if constexpr (std::is_same_v<IO, bf16_t>) {
    bf16x4 q;
#pragma unroll
    for (int r = 0; r < 4; ++r) q[r] = static_cast<__bf16>(x[r]);
    return __builtin_bit_cast(Out4<IO>, q);
  } else {
    Out4<IO> q;
#pragma unroll
    for (int r = 0; r < 4; ++r) q.e[r] = static_cast<IO>(x[r]);
    return q;
  }
}

// Log decays from a chunk's start, as two floats: their differences keep the accuracy of a small exponent.
__device__ __forceinline__ float decay(float2 to, float2 from) { return __expf((to.x - from.x) + (to.y - from.y)); }

}  // namespace sel
}  // namespace vmi
