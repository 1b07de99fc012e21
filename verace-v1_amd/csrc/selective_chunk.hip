// Chunked selective scan on the matrix cores.
//
// Over a chunk of L tokens with log decays c_t = A (d_1 + .. + d_t) from its start, S_0 the state there:
//   y_t = sum_{s<=t} (C_t . B_s) e^{c_t - c_s} d_s x_s + e^{c_t} S_0 C_t + D x_t
//   S_L = e^{c_L} S_0 + sum_s e^{c_L - c_s} d_s x_s B_s^T
// Every exponent is a difference of one chunk, so nothing overflows that the recurrence would not.
//
// Launches (Sg segments of the chunks, picked by plan()):
//   prep_kernel                d_t and c_t of every chunk (a wave each; c in fp64, kept as two floats);
//   pass_kernel<READOUT=false> (Sg > 1) each segment's own state from zero;
//   carry_kernel               (Sg > MAX_FOLD) the segments' start states;
//   pass_kernel<READOUT=true>  every segment from its start state, with outputs.
//
// A workgroup of four waves takes 64 rows p of one head and walks a segment's chunks with S^T [N, 64] in
// accumulators, 16 rows p a wave; x, B, C of the next chunk are on their way meanwhile.  S^T is directly
// the operand of S_0 C_t.  The scores of a chunk are shared: each wave forms some of the 16 x 16 tiles on
// or below the diagonal, and they pass through LDS as fragments.
// With bf16 inputs the decayed scores and the carried state enter y's products as two bf16 parts (2^-16 of a term at
// most: y is off by its own rounding and no more; one part each puts its distance to 64 bits from 1.66e-3 to 2.1e-3 and
// saves 4 of 73 us), the weighted x of the state's update as three, so the state itself is carried in fp32 throughout.
//
// Bound by instruction issue: B4 T2048 H32 P64 N128 bf16, 73 us (76 MB would move in 15).  Under the profiler, which counts
// each launch by itself: outputs 55 (of its 104k clocks a SIMD 49k issue VALU and 24k matrix instructions), own states 22.6,
// prep 5.4.  Three workgroups a compute unit.  At 256 state columns the pass with outputs spills: 44 to 50 registers in
// fp32, 2 to 4 in the 16-bit types.
#include <algorithm>

#include "selective_mfma.h"

namespace vmi {
namespace sel {

constexpr int NTH = 256;
constexpr int L = 32;        // tokens of a chunk
constexpr int PB = 64;       // rows p of a workgroup
constexpr int MAX_SEG = 64;
// Up to here a workgroup of the last pass runs over the earlier segments' states itself, from here on carry_kernel does,
// a read for each state in place of one for each pair (bf16 T2048 H32 P64 N128, carried / run over, us: 3 segments 120 /
// 114, 6 75 / 73, 8 65 / 68, 12 54 / 62).
constexpr int MAX_FOLD = 6;

struct Chunks {
  Args a;
  const float* d;            // [BH][Tp]
  const float2* c;           // [BH][Tp]
  float* seg_state;          // [Sg][BH][P][N]: a segment's own state, then (Sg > MAX_FOLD) its start state
  float* seg_decay;          // [Sg][BH]
  int nch, seg_chunks, nseg, pblocks;
  bool vec, vec_state, vec_y, fold;
};

// ------------------------------------------------------------------ step sizes and log decays
template <int LC>
__global__ __launch_bounds__(NTH) void prep_kernel(Args a, float* __restrict__ d_out, float2* __restrict__ c_out,
                                                   int nch, int64_t units) {
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (NTH / LC) + threadIdx.x / LC;
  if (unit >= units) return;
  const int l = threadIdx.x % LC;
  // heads fastest: neighbouring chunks of threads read neighbouring heads of the same tokens
  const int h = static_cast<int>(unit % a.H);
  const int64_t bc = unit / a.H;
  const int b = static_cast<int>(bc / nch), n = static_cast<int>(bc - static_cast<int64_t>(b) * nch), t = n * LC + l;
  float d = 0.f;
  double c = 0.0;
  if (t < length_of(a.lengths, a.lengths64, a.T, b)) {
    d = step_size(load_scalar(a.delta, a.delta_dtype, b * a.d_b + t * a.d_t + h) + (a.bias == nullptr ? 0.f : a.bias[h]),
                  a.softplus);
    c = static_cast<double>(d) * static_cast<double>(a.A[h]);
    // e^-10000 is 0 like e^-inf, and a chunk's sums of it stay finite: an infinite one has no differences (a NaN stays one)
    if (c < -1e4) c = -1e4;
  }
#pragma unroll
  for (int off = 1; off < LC; off <<= 1) {
    const double up = __shfl_up(c, off, LC);
    if (l >= off) c += up;
  }
  const int64_t o = (static_cast<int64_t>(b) * a.H + h) * (static_cast<int64_t>(nch) * LC) + t;
  const float hi = static_cast<float>(c);
  d_out[o] = d;
  // an infinite or NaN sum has no low part
  c_out[o] = make_float2(hi, __builtin_isfinite(hi) ? static_cast<float>(c - static_cast<double>(hi)) : 0.f);
}

// ------------------------------------------------------------------ the segments
// acc[r] += sum_{s<=t} M[t,s] x[s, r] for a chunk with values that a product with a zero does not drop.
template <typename E>
__device__ __forceinline__ void add_in_order(const E* m, int part, const E* x, int t, int l16, f32x4& acc) {
#pragma unroll 1
  for (int s = 0; s <= t; ++s) {
    float w = 0.f;
#pragma unroll
    for (int i = Parts<E>::TERM - 1; i >= 0; --i)
      w += static_cast<float>(m[i * part + (l16 + 16 * ((s >> 2) & 3)) * 8 + 4 * (s >> 4) + (s & 3)]);
    const E* row = x + Tile<E, PB>::at(s);
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] = fmaf(w, static_cast<float>(row[r]), acc[r]);
  }
}

template <typename IO, typename E, int NP, bool READOUT, bool VEC>
__global__ __launch_bounds__(NTH, sizeof(E) == 2 && NP <= 128 ? 3 : 2) void pass_kernel(Chunks k) {
  constexpr int NT = NP / 16, LT = L / 16, KN = NP / 32, NPART = Parts<E>::ALL, TERM = Parts<E>::TERM;
  typedef Tile<E, NP> TB;
  typedef Tile<E, PB> TX;
  constexpr int MS = READOUT ? LT * 64 * 8 : 8;  // a part of the scores
  __shared__ __attribute__((aligned(16))) E Bs[TB::elems(L)];
  __shared__ __attribute__((aligned(16))) E Cs[READOUT ? RowTile<E, NP>::elems(L) : 8];
  __shared__ __attribute__((aligned(16))) E Xs[TX::elems(L)];
  __shared__ __attribute__((aligned(16))) E Ms[TERM * MS];
  __shared__ __attribute__((aligned(16))) float2 cs[L];
  __shared__ __attribute__((aligned(16))) float ds[L], ws[L], es[L];
  const Args& a = k.a;
  const int tid = threadIdx.x, wave = wave_id(), lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  // neighbouring workgroups go to different XCDs: give each XCD a run of consecutive heads, which share B and C
  const uint32_t total = gridDim.x, per = total / 8, body = per * 8;
  uint32_t id = blockIdx.x;
  if (id < body) id = (id & 7) * per + (id >> 3);
  const int pb = id % k.pblocks;
  const int rest = id / k.pblocks;
  const int seg = rest / a.H % k.nseg, h = rest % a.H, b = rest / (a.H * k.nseg);
  if (!READOUT && seg == k.nseg - 1) return;  // nothing starts from its state
  const int64_t bh = static_cast<int64_t>(b) * a.H + h;
  const int p0 = pb * PB, pw = p0 + 16 * wave, grp = h / (a.H / a.G);
  const int len = length_of(a.lengths, a.lengths64, a.T, b);
  const int c0 = seg * k.seg_chunks, c1 = min(min(k.nch, c0 + k.seg_chunks), (len + L - 1) / L);
  const bool live = pw < a.P;  // this wave has rows
  const IO* x = static_cast<const IO*>(a.x) + b * a.x_b + static_cast<int64_t>(h) * a.P + p0;
  const IO* bm = static_cast<const IO*>(a.bm) + b * a.b_b + static_cast<int64_t>(grp) * a.N;
  const IO* cm = static_cast<const IO*>(a.cm) + b * a.c_b + static_cast<int64_t>(grp) * a.N;
  const int64_t tp = static_cast<int64_t>(k.nch) * L;
  const float* dp = k.d + bh * tp;
  const float2* cp = k.c + bh * tp;

  Stage<IO, E, PB, L, NTH, VEC> sx;
  Stage<IO, E, NP, L, NTH, VEC> sb, sc;
  sx.init(x, a.x_t, a.P - p0);
  sb.init(bm, a.b_t, a.N);
  if constexpr (READOUT) sc.init(cm, a.c_t, a.N);
  float rd = 0.f;
  float2 rc = make_float2(0.f, 0.f), rl = rc;
  auto fetch = [&](int c) {
    sx.fetch(c * L, len);
    sb.fetch(c * L, len);
    if constexpr (READOUT) sc.fetch(c * L, len);
    if (tid < L) {
      rd = dp[c * L + tid];
      rc = cp[c * L + tid];
      rl = cp[c * L + L - 1];
    }
  };
  if (c0 < c1) fetch(c0);

  // S^T: tile j, register r = state column n = 16 j + 4 g + r of row p = pw + l16
  f32x4 S[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) S[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  if constexpr (READOUT) {
    const int p = pw + l16;
    auto load = [&](const float* src, int j) {
      const int n = 16 * j + 4 * g;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (p >= a.P || n >= a.N) return v;
      const float* q = src + static_cast<int64_t>(p) * a.N + n;
      if (k.vec_state) return *reinterpret_cast<const f32x4*>(q);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < a.N) v[r] = q[r];
      return v;
    };
    const int64_t BH = static_cast<int64_t>(a.B) * a.H, PN = static_cast<int64_t>(a.P) * a.N;
    if ((seg == 0 || k.fold) && a.state_in != nullptr)
#pragma unroll
      for (int j = 0; j < NT; ++j) S[j] = load(a.state_in + bh * PN, j);
    // the segments before this one, or its start state alone
#pragma unroll 2
    for (int s = k.fold ? 0 : seg; s < (k.fold ? seg : seg + min(seg, 1)); ++s) {
      const float dec = k.fold ? k.seg_decay[s * BH + bh] : 0.f;
#pragma unroll
      for (int j = 0; j < NT; ++j) S[j] = S[j] * dec + load(k.seg_state + (s * BH + bh) * PN, j);
    }
  }
  if constexpr (READOUT) {  // the tile right of the diagonal stays zero
    for (int i = tid; i < TERM * MS; i += NTH) Ms[i] = static_cast<E>(0.f);
  }
  const float Dh = a.D == nullptr ? 0.f : a.D[h];
  double seg_c = 0.0;
  // where this lane's y of the chunk's first 16 tokens lies, and the way to the next 16
  const int64_t y16 = 16 * static_cast<int64_t>(a.H) * a.P;
  IO* y = static_cast<IO*>(a.y) + ((static_cast<int64_t>(b) * a.T + c0 * L + l16) * a.H + h) * a.P + pw + 4 * g;
  const bool y_on = pw + 4 * g < a.P && a.y != nullptr;

  for (int c = c0; c < c1; ++c) {
    lds_barrier();  // the last chunk's readers are done
    sx.commit(Xs);
    sb.commit(Bs);
    if constexpr (READOUT) sc.commit_rows(Cs);
    if (tid < L) {
      cs[tid] = rc;
      ds[tid] = rd;
      es[tid] = __expf(rc.x + rc.y);
      ws[tid] = rd * decay(rl, rc);
    }
    lds_barrier();
    fetch(c + 1 < c1 ? c + 1 : c);

    f32x4 acc[LT];
    if constexpr (READOUT) {
      // scores, transposed (rows s, column t): (C_t . B_s) e^{c_t - c_s} d_s
      // three tiles on or below the diagonal, one wave each
      if (wave < 3) {
        const int tt = wave != 0, st = wave == 2;
        f32x4 m = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < KN; ++kb)
          m = mma(row_frag<E, NP>(Bs, 16 * st, 32 * kb, l16, g), packed_frag<E, NP, L>(Cs, 16 * tt, 32 * kb, l16, g), m);
        const float2 ct = cs[16 * tt + l16];
        struct alignas(4 * sizeof(E)) M4 { E e[4]; } q[TERM];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int s = 16 * st + 4 * g + r;
          float v = m[r] * (decay(ct, cs[s]) * ds[s]);
          v = s <= 16 * tt + l16 ? v : 0.f;
#pragma unroll
          for (int i = 0; i < TERM; ++i) {
            q[i].e[r] = static_cast<E>(v);
            v -= static_cast<float>(q[i].e[r]);
          }
        }
#pragma unroll
        for (int i = 0; i < TERM; ++i) *reinterpret_cast<M4*>(Ms + i * MS + (tt * 64 + lane) * 8 + 4 * st) = q[i];
      }
      // S_0 C_t, transposed: rows p, column t
#pragma unroll
      for (int t = 0; t < LT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (live) {
#pragma unroll
        for (int kb = 0; kb < KN; ++kb) {
          const f32x4 s[2] = {S[2 * kb], S[2 * kb + 1]};
          Frag<E> sp[TERM], cf[LT];
          split<E>(s, sp);
#pragma unroll
          for (int t = 0; t < LT; ++t) cf[t] = packed_frag<E, NP, L>(Cs, 16 * t, 32 * kb, l16, g);
#pragma unroll
          for (int i = TERM - 1; i >= 0; --i)
#pragma unroll
            for (int t = 0; t < LT; ++t) acc[t] = mma(sp[i], cf[t], acc[t]);
        }
      }
    }
    Frag<E> xf;
    if (live) {
      xf = col_frag<E, PB>(Xs, 0, 16 * wave, l16, g);
      const float dl = es[L - 1];
#pragma unroll
      for (int j = 0; j < NT; ++j) S[j] *= dl;
      f32x4 wx[2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) wx[hf] = half(xf, hf) * *reinterpret_cast<const f32x4*>(ws + 16 * hf + 4 * g);
      Frag<E> part[NPART];
      split<E>(wx, part);
      constexpr int JB = NT < 4 ? NT : 4;  // chains in flight
#pragma unroll
      for (int j0 = 0; j0 < NT; j0 += JB) {
        Frag<E> bt[JB];
#pragma unroll
        for (int j = 0; j < JB; ++j) bt[j] = col_frag<E, NP>(Bs, 0, 16 * (j0 + j), l16, g);
#pragma unroll
        for (int q = NPART - 1; q >= 0; --q)
#pragma unroll
          for (int j = 0; j < JB; ++j) S[j0 + j] = mma(bt[j], part[q], S[j0 + j]);
      }
    }
    if constexpr (!READOUT) {
      seg_c += static_cast<double>(cs[L - 1].x) + static_cast<double>(cs[L - 1].y);
    } else {
      lds_barrier();  // the scores are in LDS
      if (live) {
#pragma unroll
        for (int t = 0; t < LT; ++t) {
          acc[t] *= es[16 * t + l16];
          f32x4 sum = acc[t];
#pragma unroll
          for (int i = TERM - 1; i >= 0; --i) {
            const E* m = Ms + i * MS + (t * 64 + lane) * 8;
            Frag<E> f;
            if constexpr (sizeof(E) == 2) {
              f.v = *reinterpret_cast<const bf16x8*>(m);
            } else {
              f.v[0] = *reinterpret_cast<const f32x4*>(m);
              f.v[1] = *reinterpret_cast<const f32x4*>(m + 4);
            }
            sum = mma(xf, f, sum);
          }
          // a NaN or an infinity in x times a masked score's 0: in order, so that no earlier token sees it
          if (__builtin_isunordered(sum[0], sum[1]) || __builtin_isunordered(sum[2], sum[3]))
            add_in_order<E>(Ms + t * 64 * 8, MS, Xs + 16 * wave + 4 * g, 16 * t + l16, l16, acc[t]);
          else
            acc[t] = sum;
          if (y_on && c * L + 16 * t + l16 < a.T) {
            const E* xr = Xs + TX::at(16 * t + l16) + 16 * wave + 4 * g;
            IO* yt = y + t * y16;
            f32x4 o;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = fmaf(Dh, static_cast<float>(xr[r]), acc[t][r]);
            if (c * L + L > len) {  // behind the length 0, whatever a NaN made of the zeros there
#pragma unroll
              for (int r = 0; r < 4; ++r) o[r] = c * L + 16 * t + l16 < len ? o[r] : 0.f;
            }
            const Out4<IO> v = out4<IO>(o);
            if (k.vec_y) {
              *reinterpret_cast<Out4<IO>*>(yt) = v;
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (pw + 4 * g + r < a.P) yt[r] = v.e[r];
            }
          }
        }
      }
      y += LT * y16;
    }
  }
  if constexpr (READOUT) {  // tokens of chunks behind the sequence's end
    if (a.y != nullptr) {
      const int z0 = max(c0, c1) * L, z1 = min(a.T, (c0 + k.seg_chunks) * L), w = min(PB, a.P - p0);
      for (int t = z0 + tid / PB; t < z1; t += NTH / PB)
        if (tid % PB < w)
          io<IO>::store(static_cast<IO*>(a.y), ((static_cast<int64_t>(b) * a.T + t) * a.H + h) * a.P + p0 + tid % PB, 0.f);
    }
  }
  float* dst = nullptr;
  if constexpr (READOUT) {
    if (seg == k.nseg - 1) dst = a.state_out + bh * a.P * a.N;
  } else {
    dst = k.seg_state + (static_cast<int64_t>(seg) * a.B * a.H + bh) * a.P * a.N;
    if (pb == 0 && tid == 0) k.seg_decay[static_cast<int64_t>(seg) * a.B * a.H + bh] = expf(static_cast<float>(seg_c));
  }
  if (dst == nullptr) return;
  const int p = pw + l16;
  if (p >= a.P) return;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int n = 16 * j + 4 * g;
    if (n >= a.N) continue;
    float* q = dst + static_cast<int64_t>(p) * a.N + n;
    if (k.vec_state) {
      *reinterpret_cast<f32x4*>(q) = S[j];
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < a.N) q[r] = S[j][r];
    }
  }
}

// seg_state[s] <- start of segment s for s >= 1, from the segments' own states: four values a thread.
__global__ __launch_bounds__(NTH) void carry_kernel(float* seg_state, const float* __restrict__ seg_decay,
                                                    const float* __restrict__ state_in, int nseg, int64_t BH, int64_t PN,
                                                    bool vec) {
  const int64_t total = BH * PN, w = vec ? 4 : 1;
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * NTH + threadIdx.x) * w;
  if (i >= total) return;
  const int64_t bh = i / PN;
  if (vec) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (state_in != nullptr) s = *reinterpret_cast<const f32x4*>(state_in + i);
    f32x4 own = *reinterpret_cast<const f32x4*>(seg_state + i);
    for (int g = 0; g + 1 < nseg; ++g) {
      s = s * seg_decay[g * BH + bh] + own;
      if (g + 2 < nseg) own = *reinterpret_cast<const f32x4*>(seg_state + (g + 1) * total + i);
      *reinterpret_cast<f32x4*>(seg_state + (g + 1) * total + i) = s;
    }
  } else {
    float s = state_in == nullptr ? 0.f : state_in[i], own = seg_state[i];
    for (int g = 0; g + 1 < nseg; ++g) {
      s = s * seg_decay[g * BH + bh] + own;
      if (g + 2 < nseg) own = seg_state[(g + 1) * total + i];
      seg_state[(g + 1) * total + i] = s;
    }
  }
}

namespace {

struct Plan {
  int64_t nch, tp, d_bytes, c_bytes, state_bytes, decay_bytes;
  int pblocks, seg_chunks, nseg;
  int64_t bytes() const { return d_bytes + c_bytes + state_bytes + decay_bytes; }
};

// Three workgroups a compute unit; a segment costs its state's way through memory, so it keeps four chunks, or two
// while every workgroup has a compute unit to itself and the chunks' own latency is what counts (fp32 N64, four / two:
// B3 T777 H8 34.7 / 29.1 us, B1 T512 H8 27.4 / 22.5; with 640 workgroups B4 T300 H32 N128 45 / 60).
Plan plan(int64_t B, int64_t T, int64_t H, int64_t P, int64_t N) {
  Plan p;
  p.nch = (T + L - 1) / L;
  p.tp = p.nch * L;
  p.pblocks = static_cast<int>((P + PB - 1) / PB);
  const int64_t base = B * H * p.pblocks, want = (768 + base - 1) / base;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(MAX_SEG, std::max(p.nch / 4, std::min(p.nch / 2, 256 / base))));
  int64_t nseg = std::min(want, most);
  p.seg_chunks = static_cast<int>((p.nch + nseg - 1) / nseg);
  p.nseg = static_cast<int>((p.nch + p.seg_chunks - 1) / p.seg_chunks);
  p.d_bytes = up16(B * H * p.tp * 4);
  p.c_bytes = up16(B * H * p.tp * 8);
  p.state_bytes = p.nseg > 1 ? up16(p.nseg * B * H * P * N * 4) : 0;
  p.decay_bytes = p.nseg > 1 ? up16(p.nseg * B * H * 4) : 0;
  return p;
}

template <typename IO, typename E, int NP, bool VEC>
int run(Chunks k, const Plan& p, hipStream_t stream) {
  const Args& a = k.a;
  const int64_t wgs = static_cast<int64_t>(a.B) * a.H * p.pblocks * p.nseg;
  const int64_t BH = static_cast<int64_t>(a.B) * a.H, PN = static_cast<int64_t>(a.P) * a.N;
  if (!grid_fits(wgs, NTH)) return VMI_ERR_UNSUPPORTED;
  if (const int st = launch_prep(a, L, const_cast<float*>(k.d), const_cast<float2*>(k.c), static_cast<int>(p.nch), stream);
      st != VMI_OK)
    return st;
  if (p.nseg > 1) {
    hipLaunchKernelGGL((pass_kernel<IO, E, NP, false, VEC>), dim3(static_cast<unsigned>(wgs)), dim3(NTH), 0, stream, k);
    if (const int st = hip_status(hipGetLastError()); st != VMI_OK) return st;
  }
  if (p.nseg > 1 && !k.fold) {
    const bool vec = PN % 4 == 0 && aligned16({a.state_in});
    const int64_t blocks = (BH * PN / (vec ? 4 : 1) + NTH - 1) / NTH;
    if (!grid_fits(blocks, NTH)) return VMI_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(carry_kernel, dim3(static_cast<unsigned>(blocks)), dim3(NTH), 0, stream, k.seg_state,
                       k.seg_decay, a.state_in, p.nseg, BH, PN, vec);
    if (const int st = hip_status(hipGetLastError()); st != VMI_OK) return st;
  }
  hipLaunchKernelGGL((pass_kernel<IO, E, NP, true, VEC>), dim3(static_cast<unsigned>(wgs)), dim3(NTH), 0, stream, k);
  return hip_status(hipGetLastError());
}

template <typename IO, typename E> int by_state(const Chunks& k, const Plan& p, hipStream_t stream) {
  auto go = [&](auto np) -> int {
    constexpr int NP = decltype(np)::value;
    return k.vec ? run<IO, E, NP, true>(k, p, stream) : run<IO, E, NP, false>(k, p, stream);
  };
  if (k.a.N <= 32) return go(std::integral_constant<int, 32>{});
  if (k.a.N <= 64) return go(std::integral_constant<int, 64>{});
  if (k.a.N <= 128) return go(std::integral_constant<int, 128>{});
  return go(std::integral_constant<int, 256>{});
}

}  // namespace

int launch_prep(const Args& a, int tokens, float* d, float2* c, int nch, hipStream_t stream) {
  const int64_t units = static_cast<int64_t>(a.B) * a.H * nch, blocks = (units + NTH / tokens - 1) / (NTH / tokens);
  if (!grid_fits(blocks, NTH)) return VMI_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (tokens == 64) hipLaunchKernelGGL(prep_kernel<64>, grid, dim3(NTH), 0, stream, a, d, c, nch, units);
  else hipLaunchKernelGGL(prep_kernel<32>, grid, dim3(NTH), 0, stream, a, d, c, nch, units);
  return hip_status(hipGetLastError());
}

// us of a call from a held state, token by token / in chunks (H32 P64 N128): bf16 B64 T4 41 / 38, T8 65 / 38; B8 T8 17 /
// 20, T12 24 / 20; B1 T12 18 / 20, T15 22 / 21.  fp32 B64 T12 71 / 57; B1 T15 19 / 20.  Many tokens' states
// make a token by token call wait on memory, so the chunks pay sooner.
bool use_chunk(int64_t B, int64_t T, int64_t H, int64_t P, int64_t N, int dtype) {
  // (segments only multiply the first where it is small)
  if (!grid_fits(B * H * ((P + PB - 1) / PB), NTH) || !grid_fits(B * H * ((T + L - 1) / L) / (NTH / L) + 1, NTH)) return false;
  return T >= (dtype == VMI_BF16 && B * H * P * N >= (1 << 22) ? 5 : 12);
}

size_t chunk_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t P, int64_t N, int dtype) {
  return use_chunk(B, T, H, P, N, dtype) ? static_cast<size_t>(plan(B, T, H, P, N).bytes()) : 0;
}

int launch_chunk(const Args& a, int dtype, void* workspace, hipStream_t stream) {
  const Plan p = plan(a.B, a.T, a.H, a.P, a.N);
  Chunks k{};
  k.a = a;
  char* w = static_cast<char*>(workspace);
  k.c = reinterpret_cast<const float2*>(w);
  k.d = reinterpret_cast<const float*>(w + p.c_bytes);
  k.seg_state = reinterpret_cast<float*>(w + p.c_bytes + p.d_bytes);
  k.seg_decay = reinterpret_cast<float*>(w + p.c_bytes + p.d_bytes + p.state_bytes);
  k.nch = static_cast<int>(p.nch), k.seg_chunks = p.seg_chunks, k.nseg = p.nseg, k.pblocks = p.pblocks;
  const int el = dtype == VMI_F32 ? 4 : 8;
  k.vec = a.P % el == 0 && a.x_t % el == 0 && a.x_b % el == 0 && a.N % el == 0 && a.b_t % el == 0 &&
          a.b_b % el == 0 && a.c_t % el == 0 && a.c_b % el == 0 && aligned16({a.x, a.bm, a.cm});
  k.vec_state = a.N % 4 == 0 && aligned16({a.state_in, a.state_out});
  k.fold = p.nseg <= MAX_FOLD;
  k.vec_y = a.P % 4 == 0 && aligned16({a.y});
  if (dtype == VMI_BF16) return by_state<bf16_t, __bf16>(k, p, stream);
  if (dtype == VMI_F16) return by_state<f16_t, float>(k, p, stream);
  return by_state<float, float>(k, p, stream);
}

}  // namespace sel
}  // namespace vmi
