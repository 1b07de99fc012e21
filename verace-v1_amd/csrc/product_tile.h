// Tiles of matrix products for gfx950: C[m][n] = sum_k A(m, k) B(n, k) with fp32 accumulators, for bf16, fp16, fp32 and
// e4m3 operands, each stored with k contiguous in a row (weights [N, K], activations [M, K]) or with m (n) contiguous
// (the same tensors in a backward pass).  The epilogue gets the accumulators.
//
// A tile has two pieces of HM rows of A and two of HN rows of B; 128 bytes of k are a step.  A step's four pieces lie in one
// of two LDS stages, filled by direct loads.  A step has two phases; a phase reads two pieces into registers, issues the loads
// of two that went free a phase ago, and multiplies A's piece with both of B's:
//
//     phase   reads                   loads                              products
//       P     A0, B1                  B0 of step t + 2, A1 of t + 1      A0 B0, A0 B1
//       Q     A1, B0 of step t + 1    A0 of step t + 2, B1 of t + 2      A1 B0, A1 B1
//
// A barrier ends the reading and the multiplying half of each phase.  With two waves a SIMD the halves of the workgroup go
// one half-phase apart, so one wave of a SIMD multiplies while the other reads (STAGGER).  A wave waits for its own loads
// of a piece at the end of the reading half before the one that reads it, one barrier ahead of every reader, with the four
// pieces issued later still in flight.
//
// For few tiles of a long contraction several groups of a tile's waves take a share of the steps each, with two LDS stages of
// their own, and add their sums through LDS in a fixed order (join_groups).
//
// LDS is read at 16 bytes a lane (k contiguous), by transposing reads of 8 (m contiguous, 16 bits) or 4 bytes a lane (fp32),
// and its 16-byte slots are permuted so that the lanes of an access fall in distinct banks.  The direct loads write LDS in
// lane order, so the permutation is made by the addresses that they read.  Loads outside the operands return zeros: their
// offset lies beyond the buffer's size.
// The matrix cores bound long contractions (bf16, 8192 x 16384 x 4096, k contiguous in one operand: 740 us, 1.49 PFLOP/s, the
// cores busy 83 % of the time at the 1.7 GHz that the power limit leaves; e4m3 8192 x 8192 x 4096 211 us, 2.6 PFLOP/s); with
// tiles of 256 x 128 LDS does, 1408 clocks of it for 1024 of products a step (fp16, 8192 x 2048 x 1024: 45 us, 760 TFLOP/s).
#pragma once

#include "vmi_common.h"
#include "vmi_mfma.h"

namespace vmi {
namespace prod {

struct e4m3 {
  uint8_t bits;
};
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

// Sixteen rows of each operand over 128 bytes of k: lane l holds row l % 16, and of each half (64 bytes) the 16 bytes at
// 16 * (l / 16) (fp32: every fourth k of them).  The order of k is the same in both operands and otherwise free.
typedef i32x8 Frag;

template <typename E> __device__ __forceinline__ f32x4 mma(Frag b, Frag a, f32x4 c);
template <> __device__ __forceinline__ f32x4 mma<__bf16>(Frag b, Frag a, f32x4 c) {
  c = mfma_t<__bf16>::mma16(__builtin_bit_cast(bf16x8, (i32x4)b.lo), __builtin_bit_cast(bf16x8, (i32x4)a.lo), c);
  return mfma_t<__bf16>::mma16(__builtin_bit_cast(bf16x8, (i32x4)b.hi), __builtin_bit_cast(bf16x8, (i32x4)a.hi), c);
}
template <> __device__ __forceinline__ f32x4 mma<_Float16>(Frag b, Frag a, f32x4 c) {
  c = mfma_t<_Float16>::mma16(__builtin_bit_cast(f16x8, (i32x4)b.lo), __builtin_bit_cast(f16x8, (i32x4)a.lo), c);
  return mfma_t<_Float16>::mma16(__builtin_bit_cast(f16x8, (i32x4)b.hi), __builtin_bit_cast(f16x8, (i32x4)a.hi), c);
}
template <> __device__ __forceinline__ f32x4 mma<float>(Frag b, Frag a, f32x4 c) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, (int)b[e]), __builtin_bit_cast(float, (int)a[e]), c, 0, 0, 0);
  return c;
}
// The instruction takes eight consecutive products of a sum on one scale: each is cut toward 0 to a multiple of 2^-13 of the power of
// two of the largest before they add up, in fp32 with the other eights' (the 16x16x32 8-bit instruction likewise).  Of 128 normal
// values that is 2e-6 rms of the sum's magnitudes, 9.5e-6 at most seen: far below the operands' own four bits and half a step of a
// 16-bit result.  Exact products would take both operands through 16 bits, at half the rate and a conversion of each.
template <> __device__ __forceinline__ f32x4 mma<e4m3>(Frag b, Frag a, f32x4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, 0, 0, 0, 0, 0, 0);  // both e4m3, no block scales
}

constexpr unsigned kOutside = 0x80000000u;  // an offset past every buffer

__device__ __forceinline__ unsigned lds_offset(const void* p) {
  return static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)(p)));
}
// 64 lanes x 16 bytes from base + off straight into LDS at `lds` (the wave's, uniform), zeros where off is kOutside.  As an
// asm block so that the compiler adds no waits of its own around LDS reads; it has no register results.
__device__ __forceinline__ void load_lds(const char* base, unsigned off, unsigned lds) {
  const uint64_t b = reinterpret_cast<uint64_t>(base);
  const i32x4 srd = {static_cast<int>(b), static_cast<int>(b >> 32), static_cast<int>(kOutside - 16), 0x20000};
  asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"{m0}"(lds), "v"(off), "s"(srd) : "memory");
}
template <int N> __device__ __forceinline__ void wait_loads_and_lds() {
  static_assert(N < 64);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14));  // vmcnt(N), lgkmcnt(0)
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// HM, HN: rows of a piece; WM x WN waves, each with MF x NF fragments of 16 x 16 of each of the four products.
template <int HM_, int HN_, int WM_, int WN_> struct Shape {
  static constexpr int HM = HM_, HN = HN_, WM = WM_, WN = WN_, THREADS = 64 * WM * WN;
  static constexpr int MF = HM / (16 * WM), NF = HN / (16 * WN);
  static constexpr int LA = HM * 8 / THREADS, LB = HN * 8 / THREADS;  // loads of a thread for a piece
  static constexpr int A_BYTES = HM * 128, B_BYTES = HN * 128, STAGE = 2 * (A_BYTES + B_BYTES);
  static constexpr int FLIGHT = 2 * (LA + LB);  // the loads of four pieces
  static constexpr bool STAGGER = WM * WN == 8;
  static_assert(LA >= 1 && LB >= 1 && MF >= 1 && NF >= 1);
};

// A thread's loads of one piece of an operand, `MN` where its m (n) is contiguous in memory.  H rows (columns) of the piece, of
// which `inside` are in the operand.
// PERM: the order in which B's columns go to fragments (see column_of).
template <typename E, bool MN, int H, int L, int THREADS, int XF, bool PERM> struct Loader {
  static constexpr int SIZE = sizeof(E), KT = 128 / SIZE, RB = MN ? H * SIZE : 128, SLOTS = RB / 16;
  unsigned off[L];
  int k[L];  // the first k of the load within a step, in elements

  __device__ __forceinline__ static int swizzle(int row) {
    if constexpr (!MN) return (row >> 1) & 7;
    else if constexpr (SIZE == 4) return ((row >> 2) & (SLOTS >= 16 ? 3 : 1)) << 2;
    else if constexpr (SLOTS >= 16) return ((row & 3) << 2) | (((row >> 3) & 1) << 1);
    else if constexpr (SLOTS == 8) return (((row >> 1) & 1) | (((row >> 3) & 1) << 1)) << 1;
    else return ((row >> 3) & 1) << 1;
  }
  __device__ __forceinline__ void init(int tid, unsigned ld, int inside) {
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int c = i * THREADS + tid, row = c / SLOTS, slot = (c % SLOTS) ^ swizzle(row);
      if constexpr (MN) {
        const int x = slot * (16 / SIZE);
        k[i] = row;
        off[i] = x < inside ? row * ld + slot * 16 : kOutside;
      } else {
        int x = row;
        if constexpr (PERM) {
          const int r = row % (16 * XF), j = r / 16, q = r % 16;
          x = row - r + (q / 4) * 4 * XF + j * 4 + q % 4;
        }
        k[i] = slot * (16 / SIZE);
        off[i] = x < inside ? x * ld + slot * 16 : kOutside;
      }
    }
  }
  // left: how many k there are from the step's first on
  __device__ __forceinline__ void issue(const char* base, int left, unsigned lds) const {
#pragma unroll
    for (int i = 0; i < L; ++i) load_lds(base, k[i] < left ? off[i] : kOutside, lds + i * THREADS * 16);
  }
};

// Reads XF fragments of a piece; `first`: the wave's first row (column) of the piece.
template <typename E, bool MN, int H, int XF> struct Reader {
  static constexpr int SIZE = sizeof(E), RB = H * SIZE;
  unsigned at[MN ? XF : 2];
  __device__ __forceinline__ void init(int lane, int first) {
    const int i = lane & 15, q = lane >> 4;
    if constexpr (!MN) {
      const int x = (i >> 1) & 7;
      at[0] = (first + i) * 128 + ((q ^ x) << 4);
      at[1] = at[0] ^ 64;
    } else if constexpr (SIZE == 2) {
      // lane 4 e + p of a group of 16 addresses row k = 8 q + e and the 4 columns at 4 p
      const int e = i >> 2, p = i & 3, k = 8 * q + e;
#pragma unroll
      for (int f = 0; f < XF; ++f) {
        const int c4 = (first + f * 16) / 4 + p;
        at[f] = k * RB + (((c4 >> 1) ^ Loader<E, MN, H, 1, 64, 1, false>::swizzle(k)) << 4) + (c4 & 1) * 8;
      }
    } else {
#pragma unroll
      for (int f = 0; f < XF; ++f) {
        const int c = first + f * 16 + i;
        at[f] = 4 * q * RB + (((c >> 2) ^ Loader<E, MN, H, 1, 64, 1, false>::swizzle(4 * q)) << 4) + (c & 3) * 4;
      }
    }
  }
  __device__ __forceinline__ void read(const char* piece, Frag (&f)[XF]) const {
    if constexpr (!MN) {
#pragma unroll
      for (int x = 0; x < XF; ++x) {
        f[x].lo = *reinterpret_cast<const i32x4*>(piece + at[0] + x * 2048);
        f[x].hi = *reinterpret_cast<const i32x4*>(piece + at[1] + x * 2048);
      }
    } else if constexpr (SIZE == 2) {
#pragma unroll
      for (int x = 0; x < XF; ++x) {
        i16x4 v[4];
#pragma unroll
        for (int h = 0; h < 4; ++h)  // k + 32 * (h / 2) + 4 * (h % 2)
          v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_i16x4*)(piece + at[x] + (32 * (h / 2) + 4 * (h % 2)) * RB));
        typedef short i16x8 __attribute__((ext_vector_type(8)));
        f[x].lo = __builtin_bit_cast(i32x4, (i16x8)__builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
        f[x].hi = __builtin_bit_cast(i32x4, (i16x8)__builtin_shufflevector(v[2], v[3], 0, 1, 2, 3, 4, 5, 6, 7));
      }
    } else {
#pragma unroll
      for (int x = 0; x < XF; ++x)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          f[x][e] = *reinterpret_cast<const int*>(piece + at[x] + ((e / 4) * 16 + e % 4) * RB);
    }
  }
};

// A tile's operands: two pieces of A and two of B at their first k, and (SEGMENTS == 2) again the second part of k.
struct Operands {
  const char* a[2];
  const char* b[2];
  int64_t a_step, b_step;    // bytes from one step of k to the next
  unsigned lda, ldb;         // bytes
  int a_inside[2], b_inside[2];
  int k;                     // elements of k (of each segment)
  const char* a2[2];
  const char* b2[2];
};

template <typename S> struct Acc {
  f32x4 v[2][2][S::MF][S::NF];
};

// GROUPS: that many groups of S::THREADS threads have a share of k and two LDS stages each.
template <typename E, bool AMN, bool BMN, typename S, int SEGMENTS, int GROUPS>
__device__ __forceinline__ void tile_product(Operands& o, char* lds, Acc<S>& acc) {
  constexpr int KT = 128 / sizeof(E);
  constexpr bool PERM = !BMN, STAGGER = S::STAGGER || GROUPS > 1;
  const int tid = threadIdx.x % S::THREADS, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = GROUPS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / S::THREADS);
  const bool late = STAGGER && __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) >= S::THREADS * GROUPS / 128;
  lds += group * 2 * S::STAGE;
  const int wm = wave / S::WN, wn = wave % S::WN;
  Loader<E, AMN, S::HM, S::LA, S::THREADS, S::MF, false> la[2];
  Loader<E, BMN, S::HN, S::LB, S::THREADS, S::NF, PERM> lb[2];
  Reader<E, AMN, S::HM, S::MF> ra;
  Reader<E, BMN, S::HN, S::NF> rb;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    la[h].init(tid, o.lda, o.a_inside[h]);
    lb[h].init(tid, o.ldb, o.b_inside[h]);
  }
  ra.init(lane, wm * 16 * S::MF);
  rb.init(lane, wn * 16 * S::NF);
  const int steps = (o.k + KT * GROUPS - 1) / (KT * GROUPS), total = SEGMENTS * steps, before = group * steps;
  const int k_left = o.k - before * KT;  // may be none
  const unsigned lds_wave = lds_offset(lds) + wave * 1024;
  // pieces of a stage: B0, A0, B1, A1, the order of their loads
  constexpr int at_b[2] = {0, S::B_BYTES + S::A_BYTES}, at_a[2] = {S::B_BYTES, 2 * S::B_BYTES + S::A_BYTES};
  const char* pa[2] = {o.a[0] + before * o.a_step, o.a[1] + before * o.a_step};
  const char* pb[2] = {o.b[0] + before * o.b_step, o.b[1] + before * o.b_step};
  auto left = [&](int t) { return k_left - (SEGMENTS == 2 && t >= steps ? t - steps : t) * KT; };
  auto issue_a = [&](int h, int t) {
    if (SEGMENTS == 2 && t == steps) pa[h] = o.a2[h] + before * o.a_step;
    la[h].issue(pa[h], t < total ? left(t) : 0, lds_wave + (t & 1) * S::STAGE + at_a[h]);
    pa[h] += o.a_step;
  };
  auto issue_b = [&](int h, int t) {
    if (SEGMENTS == 2 && t == steps) pb[h] = o.b2[h] + before * o.b_step;
    lb[h].issue(pb[h], t < total ? left(t) : 0, lds_wave + (t & 1) * S::STAGE + at_b[h]);
    pb[h] += o.b_step;
  };
#pragma unroll
  for (int hm = 0; hm < 2; ++hm)
#pragma unroll
    for (int hn = 0; hn < 2; ++hn)
#pragma unroll
      for (int m = 0; m < S::MF; ++m)
#pragma unroll
        for (int n = 0; n < S::NF; ++n) acc.v[hm][hn][m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  Frag a[S::MF], b0[S::NF], b0_next[S::NF], b1[S::NF];
  auto multiply = [&](f32x4 (&c0)[S::MF][S::NF], f32x4 (&c1)[S::MF][S::NF], const Frag (&x0)[S::NF]) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int m = 0; m < S::MF; ++m)
#pragma unroll
      for (int n = 0; n < S::NF; ++n) c0[m][n] = mma<E>(x0[n], a[m], c0[m][n]);
#pragma unroll
    for (int m = 0; m < S::MF; ++m)
#pragma unroll
      for (int n = 0; n < S::NF; ++n) c1[m][n] = mma<E>(b1[n], a[m], c1[m][n]);
    __builtin_amdgcn_s_setprio(0);
  };
  auto step = [&](int t, Frag (&x0)[S::NF], Frag (&x0_next)[S::NF]) {
    const char* st = lds + (t & 1) * S::STAGE;
    ra.read(st + at_a[0], a);
    rb.read(st + at_b[1], b1);
    issue_b(0, t + 2);
    issue_a(1, t + 1);
    wait_loads_and_lds<S::FLIGHT>();
    barrier();
    multiply(acc.v[0][0], acc.v[0][1], x0);
    barrier();
    ra.read(st + at_a[1], a);
    rb.read(lds + ((t + 1) & 1) * S::STAGE + at_b[0], x0_next);
    issue_a(0, t + 2);
    issue_b(1, t + 2);
    wait_loads_and_lds<S::FLIGHT>();
    barrier();
    multiply(acc.v[1][0], acc.v[1][1], x0);
    barrier();
  };
  issue_b(0, 0);
  issue_a(0, 0);
  issue_b(1, 0);
  issue_b(0, 1);
  issue_a(1, 0);
  issue_a(0, 1);
  issue_b(1, 1);
  wait_loads_and_lds<S::FLIGHT>();
  barrier();
  rb.read(lds + at_b[0], b0);
  wait_loads_and_lds<S::FLIGHT>();
  barrier();
  if (STAGGER && late) barrier();
  int t = 0;
  for (; t + 1 < total; t += 2) {
    step(t, b0, b0_next);
    step(t + 1, b0_next, b0);
  }
  if (t < total) step(t, b0, b0_next);
  if (STAGGER && !late) barrier();
  wait_loads_and_lds<0>();  // no load may write LDS after the workgroup's end
}

// The groups' sums of a tile added, in order: group g gets the part (hm, hn) = (g % 2, HNS == 1 ? g / 2 : 0 and 1) in v[0].
template <typename S, int GROUPS, int HNS> __device__ __forceinline__ void join_groups(char* lds, Acc<S>& acc) {
  constexpr int EACH = S::MF * S::NF * S::THREADS, PART = 4 * EACH;
  static_assert(PART * 16 <= 2 * S::STAGE);
  const int tid = threadIdx.x % S::THREADS, group = threadIdx.x / S::THREADS;
  __syncthreads();  // the last loads of every wave are in
#pragma unroll
  for (int hm = 0; hm < 2; ++hm)
#pragma unroll
    for (int hn = 0; hn < 2; ++hn)
#pragma unroll
      for (int f = 0; f < S::MF * S::NF; ++f)
        *reinterpret_cast<f32x4*>(lds + group * 2 * S::STAGE + ((2 * hm + hn) * EACH + f * S::THREADS + tid) * 16) =
            acc.v[hm][hn][f / S::NF][f % S::NF];
  __syncthreads();
  const int hm = group & 1, hn0 = HNS == 1 ? group >> 1 & 1 : 0;
#pragma unroll
  for (int hn = 0; hn < HNS; ++hn)
#pragma unroll
    for (int f = 0; f < S::MF * S::NF; ++f) {
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
        sum += *reinterpret_cast<const f32x4*>(lds + g * 2 * S::STAGE + ((2 * hm + hn0 + hn) * EACH + f * S::THREADS + tid) * 16);
      acc.v[0][hn][f / S::NF][f % S::NF] = sum;
    }
}

// The first of the 4 (PERM: 4 * NF over all of a wave's fragments) consecutive columns of a lane's accumulator n.
template <typename S, bool PERM> __device__ __forceinline__ int column_of(int wn, int lane, int n) {
  const int g = lane >> 4;
  return wn * 16 * S::NF + (PERM ? g * 4 * S::NF + n * 4 : n * 16 + g * 4);
}

// A workgroup's tile: eight XCDs take workgroups in turn, so each gets a run of neighbouring tiles (its own L2 then holds
// their operands), in columns of up to `GROUP` rows of tiles.
__device__ __forceinline__ void tile_of(int block, int tiles_m, int tiles_n, int group, int& tm, int& tn) {
  const int n = tiles_m * tiles_n, xcd = block & 7, i = block >> 3, each = n >> 3, rest = n & 7;
  const int t = xcd * each + (xcd < rest ? xcd : rest) + i;
  const int per = group * tiles_n, first = t / per * group, rows = tiles_m - first < group ? tiles_m - first : group;
  tm = first + (t % per) % rows;
  tn = (t % per) / rows;
}

}  // namespace prod
}  // namespace vmi
