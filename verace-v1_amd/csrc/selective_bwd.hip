// Backward of the selective scan, in chunks on the matrix cores.
//
// With G_t the gradient of S_t from everything after t and dy_t, over a chunk of L tokens with log decays c_t
// from its start, S_0 the state at its start, G_L the gradient of the state at its end, and
// dec[t,s] = e^{c_t - c_s} for s <= t:
//   Q[t,s] = (dy_t . x_s) dec d_s,   M[t,s] = (C_t . B_s) dec d_s,   R[t,s] = (C_t . B_s)(dy_t . x_s) dec
//   dC_t = sum_s Q[t,s] B_s + e^{c_t} S_0^T dy_t
//   dB_s = sum_t Q[t,s] C_t + e^{c_L - c_s} d_s G_L^T x_s
//   dx_s = sum_t M[t,s] dy_t + e^{c_L - c_s} d_s G_L B_s + D dy_s
//   G_0  = e^{c_L} G_L + sum_t e^{c_t} dy_t C_t^T
// The gradient of token t's log decay collects every path that crosses it, from s < t (or S_0) to u >= t (or
// G_L); with alpha_u = e^{c_u} dy_u . S_0 C_u, beta_s = e^{c_L - c_s} x_s . G_L B_s, kappa = e^{c_L} <G_L, S_0>:
//   g_t = kappa + sum_{u>=t} alpha_u + sum_{s<t} d_s beta_s + sum_{u>=t, s<t} R[u,s] d_s
//   dd_t = sum_u R[u,t] + beta_t + A g_t,   dA = sum d_t g_t,   ddelta = dd softplus'(.)
// Each chunk starts from its own kappa, so nothing is accumulated over the sequence but G itself.  The double sum is
// formed as it stands, tile by tile (16 x 16): as running differences of R's row and column sums it would carry every
// rounding back over the chunk (B4 T2048 H32 P64 N128, decays up to e^-1.6 a token: dbias off by 2.2e-6 of its norm
// that way, 1.3e-7 this way, at 5 us).
//
// Launches:
//   prep (selective_chunk.hip), states_kernel<OWN> and starts_kernel (more than one segment), states_kernel: the S_0
//     and G_L of every chunk, both directions in one grid, in the order in which the main kernel's fragments read them;
//   main_kernel: a workgroup of eight waves per chunk and block of heads of a group walks the heads with dB and
//     dC of the chunk in accumulators (they are sums over the heads: as partials of each head they would be the
//     largest thing moved); C . B, the same for every head, is formed once;
//   steps_kernel: g, and from it ddelta and the chunks' shares of dA and dbias;
//   reduce_kernel: the head blocks' dB and dC and the heads' dA, dD, dbias, in a fixed order.
//
// bf16 inputs: Q and M, and G_L where it enters dx, are two bf16 parts (2^-16 of a term: dx, dB and dC are off by their
// own rounding and no more; one part each saves 25 us below and puts their distance to 64 bits from 1.66e-3 to 2.3e-3);
// S_0 and G_L enter alpha, beta, dB and dC as three bf16 parts and R stays fp32, because ddelta, dA and dbias may be
// fp32 and are sums in which such roundings do not cancel.
//
// B4 T2048 H32 P64 N128 bf16, us: main 143 (one workgroup a compute unit, two waves a SIMD: of 303k clocks VALU 115k, matrix
// 50k; LDS 124k a compute unit, 44k of them bank conflicts), states 78 (268 MB of S_0 and G_L written: 57 at the copy rate),
// steps 7.6, prep 6.2, reduce 5.7.  A chunk of 64 halves the states' traffic against 32; above 128 state columns its
// accumulators and parts fit neither the registers nor LDS (193 spilled registers with one part; 5 in chunks of 32), so
// there it is 32 (forward and backward at B2 T2048 H32 P64 N256 482 us for 504).
#include <algorithm>
#include <type_traits>

#include "selective_mfma.h"

namespace vmi {
namespace sel {

constexpr int PB = 64;
constexpr int SNT = 256;     // threads of the state passes
constexpr int MNT = 512;     // and of the main kernel
constexpr int BWD_MAX_SEG = 32;

struct Bwd {
  Args a;
  const void* dy;
  int64_t y_t, y_b;
  const float* dstate;       // [B, H, P, N] or null
  const float* d;            // [BH][Tp]
  const float2* c;           // [BH][Tp]
  float* own;                // [2][Sg][BH pblocks][NP 64]: segments' own states, then their starts
  float *s0, *g1;            // [BH pblocks][nch][NP 64], tiles of 16 x 16 in fragment order
  float *pb, *pc;            // [hblocks][B T][G][N] (null: dB, dC written directly)
  float* ph;                 // [3][B nch][H]: dA, dD, dbias
  float* tok;                // [4][BH pblocks][Tp]: alpha, beta, g's sum of R d, sum_u R[u, t]
  float* chk;                // [2][BH pblocks][nch]: kappa, sum of x . dy
  void *dx, *ddelta, *db, *dc;
  float *dA, *dD, *dbias, *dstate_in;
  int nch, seg_chunks, nseg, pblocks, hblocks, hper;
  const float* Dz;           // D, or anything as long without one
  bool vec, vec_dx, has_d;
};

// ------------------------------------------------------------------ S_0 and G_L of every chunk
// Four waves, 16 rows p each: tile j, register r = row p0 + 16 wave + 4 g + r, column n = 16 j + l16.  Forward:
// S += (d_s e^{c_L - c_s} x_s) B_s^T; reverse, chunks from the last: G += (e^{c_t} dy_t) C_t^T.
template <typename IO, typename E, int NP, int L, bool OWN, bool VEC>
__global__ __launch_bounds__(SNT, 2) void states_kernel(Bwd k) {
  constexpr int NT = NP / 16, KB = L / 32, NPART = Parts<E>::ALL;
  typedef Tile<E, NP> TB;
  typedef Tile<E, PB> TX;
  __shared__ __attribute__((aligned(16))) E Bs[TB::elems(L)];
  __shared__ __attribute__((aligned(16))) E Xs[TX::elems(L)];
  __shared__ __attribute__((aligned(16))) float ws[L];
  __shared__ float wl;
  const Args& a = k.a;
  const int tid = threadIdx.x, wave = wave_id(), lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const bool reverse = blockIdx.y != 0;
  const int pb = blockIdx.x % k.pblocks, rest = blockIdx.x / k.pblocks;
  // segments in the direction's order: seg 0 is the one with the given start
  const int h = rest % a.H, seg = rest / a.H % k.nseg, b = rest / (a.H * k.nseg);
  if (OWN && seg == k.nseg - 1) return;
  const int64_t bh = static_cast<int64_t>(b) * a.H + h, bhp = bh * k.pblocks + pb;
  const int64_t BHP = static_cast<int64_t>(a.B) * a.H * k.pblocks;
  const int p0 = pb * PB, grp = h / (a.H / a.G);
  const int len = length_of(a.lengths, a.lengths64, a.T, b);
  const int place = reverse ? k.nseg - 1 - seg : seg;
  const int first = place * k.seg_chunks, last = min(min(k.nch, first + k.seg_chunks), (len + L - 1) / L);
  const int count = max(0, last - first);
  const IO* x = static_cast<const IO*>(reverse ? k.dy : a.x) + b * (reverse ? k.y_b : a.x_b) + static_cast<int64_t>(h) * a.P + p0;
  const IO* bm = static_cast<const IO*>(reverse ? a.cm : a.bm) + b * (reverse ? a.c_b : a.b_b) + static_cast<int64_t>(grp) * a.N;
  const int64_t x_t = reverse ? k.y_t : a.x_t, b_t = reverse ? a.c_t : a.b_t;
  const int64_t tp = static_cast<int64_t>(k.nch) * L;
  const float* dp = k.d + bh * tp;
  const float2* cp = k.c + bh * tp;

  Stage<IO, E, PB, L, SNT, VEC> sx;
  Stage<IO, E, NP, L, SNT, VEC> sb;
  sx.init(x, x_t, a.P - p0);
  sb.init(bm, b_t, a.N);
  float rd = 0.f;
  float2 rc = make_float2(0.f, 0.f), rl = rc;
  auto chunk = [&](int i) { return reverse ? last - 1 - i : first + i; };
  auto fetch = [&](int c) {
    sx.fetch(c * L, len);
    sb.fetch(c * L, len);
    if (tid < L) {
      rd = dp[c * L + tid];
      rc = cp[c * L + tid];
      rl = cp[c * L + L - 1];
    }
  };
  if (count > 0) fetch(chunk(0));

  f32x4 S[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) S[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (!OWN) {
    if (seg > 0) {
      const float* src = k.own + ((reverse ? k.nseg : 0) + seg) * BHP * (NP * PB) + bhp * (NP * PB);
#pragma unroll
      for (int j = 0; j < NT; ++j) S[j] = *reinterpret_cast<const f32x4*>(src + ((j * 4 + wave) * 64 + lane) * 4);
    } else {
      const float* src = reverse ? k.dstate : a.state_in;
      if (src != nullptr) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int p = p0 + 16 * wave + 4 * g + r, n = 16 * j + l16;
            if (p < a.P && n < a.N) S[j][r] = src[(bh * a.P + p) * a.N + n];
          }
      }
    }
  }
  for (int i = 0; i < count; ++i) {
    const int c = chunk(i);
    if (!OWN) {
      float* dst = (reverse ? k.g1 : k.s0) + (bhp * k.nch + c) * (NP * PB);
#pragma unroll
      for (int j = 0; j < NT; ++j) *reinterpret_cast<f32x4*>(dst + ((j * 4 + wave) * 64 + lane) * 4) = S[j];
    }
    lds_barrier();
    sx.commit(Xs);
    sb.commit(Bs);
    if (tid < L) {
      ws[tid] = reverse ? __expf(rc.x + rc.y) : rd * decay(rl, rc);
      if (tid == L - 1) wl = __expf(rc.x + rc.y);
    }
    lds_barrier();
    if (i + 1 < count) fetch(chunk(i + 1));
    const float dl = wl;
#pragma unroll
    for (int j = 0; j < NT; ++j) S[j] *= dl;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const Frag<E> xf = col_frag<E, PB>(Xs, 32 * kb, 16 * wave, l16, g);
      f32x4 wx[2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
        wx[hf] = half(xf, hf) * *reinterpret_cast<const f32x4*>(ws + 32 * kb + 16 * hf + 4 * g);
      Frag<E> part[NPART];
      split<E>(wx, part);
#pragma unroll
      for (int j0 = 0; j0 < NT; j0 += 4) {  // four chains in flight
        Frag<E> bt[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) bt[j] = col_frag<E, NP>(Bs, 32 * kb, 16 * (j0 + j), l16, g);
#pragma unroll
        for (int q = NPART - 1; q >= 0; --q)
#pragma unroll
          for (int j = 0; j < 4; ++j) S[j0 + j] = mma(part[q], bt[j], S[j0 + j]);
      }
    }
  }
  if (OWN) {
    float* dst = k.own + ((reverse ? k.nseg : 0) + seg) * BHP * (NP * PB) + bhp * (NP * PB);
#pragma unroll
    for (int j = 0; j < NT; ++j) *reinterpret_cast<f32x4*>(dst + ((j * 4 + wave) * 64 + lane) * 4) = S[j];
    return;
  }
  if (!reverse || seg != k.nseg - 1 || k.dstate_in == nullptr) return;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int p = p0 + 16 * wave + 4 * g + r, n = 16 * j + l16;
      if (p < a.P && n < a.N) k.dstate_in[(bh * a.P + p) * a.N + n] = S[j][r];
    }
}

// own[dir][s] <- start of the direction's segment s >= 1.  The decay of a segment is the same both ways; the
// given starts are read in the state's layout.
template <int NP>
__global__ __launch_bounds__(SNT) void starts_kernel(Bwd k, int L) {
  constexpr int SZ = NP * PB;
  const Args& a = k.a;
  const bool reverse = blockIdx.y != 0;
  const int64_t BHP = static_cast<int64_t>(a.B) * a.H * k.pblocks;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * SNT + threadIdx.x;  // 16-byte piece
  if (id >= BHP * (SZ / 4)) return;  // whole workgroups: SZ / 4 is a multiple of SNT
  static_assert(SZ / 4 % SNT == 0, "");
  const int64_t bhp = id / (SZ / 4);
  const int e = static_cast<int>(id - bhp * (SZ / 4)), lane = e & 63, wave = (e >> 6) & 3, j = e >> 8;
  const int64_t bh = bhp / k.pblocks;
  const int pb = static_cast<int>(bhp - bh * k.pblocks);
  const float* src = reverse ? k.dstate : a.state_in;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (src != nullptr)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int p = pb * PB + 16 * wave + 4 * (lane >> 4) + r, n = 16 * j + (lane & 15);
      if (p < a.P && n < a.N) s[r] = src[(bh * a.P + p) * a.N + n];
    }
  const int64_t tp = static_cast<int64_t>(k.nch) * L;
  const float2* cp = k.c + bh * tp;
  float* base = k.own + (reverse ? k.nseg : 0) * BHP * SZ + bhp * SZ + e * 4;
  f32x4 own = *reinterpret_cast<const f32x4*>(base);
  for (int g = 0; g + 1 < k.nseg; ++g) {
    const int place = reverse ? k.nseg - 1 - g : g;
    double c = 0.0;  // the same in all lanes: a wave's pieces are of one state
    for (int i = place * k.seg_chunks + lane; i < min(k.nch, (place + 1) * k.seg_chunks); i += 64) {
      const float2 v = cp[static_cast<int64_t>(i) * L + L - 1];
      c += static_cast<double>(v.x) + static_cast<double>(v.y);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) c += __shfl_xor(c, off);
    s = s * expf(static_cast<float>(c)) + own;
    if (g + 2 < k.nseg) own = *reinterpret_cast<const f32x4*>(base + (g + 1) * BHP * SZ);
    *reinterpret_cast<f32x4*>(base + (g + 1) * BHP * SZ) = s;
  }
}

// ------------------------------------------------------------------ the chunks
// Tile i on or below the diagonal, row by row from the last: tiles 0 .. LT - 1 are the last t-tile's.
template <int LT> __device__ __forceinline__ bool lower_tile(int i, int& tt, int& st) {
  tt = LT - 1;
#pragma unroll
  for (int r = LT; r >= 1; --r) {
    if (i < r) {
      st = i;
      return true;
    }
    i -= r;
    --tt;
  }
  return false;
}

template <typename IO, typename E, int NP, int L, bool VEC>
__global__ __launch_bounds__(MNT) void main_kernel(Bwd k) {
  constexpr int NW = MNT / 64, NT = NP / 16, LT = L / 16, KL = L / 32, KN = NP / 32, KP = PB / 32, NPART = Parts<E>::ALL, TERM = Parts<E>::TERM;
  constexpr int NTW = NT >= NW ? NT / NW : 1;      // n-tiles of a wave: wave, wave + 8 (or wave % NT)
  constexpr int TS = NT >= NW ? 1 : NW / NT;       // waves that share an n-tile, each LTW of the t-tiles
  constexpr int LTW = LT / TS;
  constexpr int GR = NP < 128 / TERM ? NP : 128 / TERM, NH = NP / GR;  // dx takes G_L through LDS GR state columns at a time
  constexpr int PER = (LT * (LT + 1) / 2 + NW - 1) / NW;
  static_assert(LT % TS == 0, "");
  typedef Tile<E, NP> TB;
  typedef Tile<E, PB> TX;
  typedef Tile<E, L> TQ;
  constexpr int QE = TQ::elems(L), GE = TX::elems(GR);
  __shared__ __attribute__((aligned(16))) E Bs[TB::elems(L)];
  __shared__ __attribute__((aligned(16))) E Cs[TB::elems(L)];
  // x, dy and the log decays of a unit while the next one's arrive
  constexpr bool XROWS = NP <= 128 || sizeof(E) == 2;  // x by lane group (12 KB of 10); where LDS is full, not
  __shared__ __attribute__((aligned(16))) E Xb[2][XROWS ? RowTile<E, PB>::elems(L) : TX::elems(L)];
  __shared__ __attribute__((aligned(16))) E Yb[2][TX::elems(L)];
  __shared__ __attribute__((aligned(16))) float2 cb2[2][L];
  __shared__ __attribute__((aligned(16))) float db2[2][L], eb2[2][L], wb2[2][L], dh2[2];
  __shared__ __attribute__((aligned(16))) E Qs[TERM * QE];            // [t][s], part by part
  __shared__ __attribute__((aligned(16))) E Ms[TERM * QE];
  __shared__ __attribute__((aligned(16))) E Gs[TERM * GE];            // G_L^T [n][p]
  __shared__ float row_r[LT][L], col_r[LT][L];                  // sums of R d_s (below) by s-tile, sum_t R by t-tile
  __shared__ float alpha[NW][L], beta[NW][L], kappa[NW], diag[LT];
  const Args& a = k.a;
  const int tid = threadIdx.x, wave = wave_id(), lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int hb = blockIdx.x % k.hblocks;
  int rest = blockIdx.x / k.hblocks;
  const int grp = rest % a.G;
  rest /= a.G;
  const int c = rest % k.nch, b = rest / k.nch;
  const int hg = a.H / a.G, h0 = grp * hg + hb * k.hper, h1 = min((grp + 1) * hg, h0 + k.hper);
  const int len = length_of(a.lengths, a.lengths64, a.T, b), t0 = c * L;
  const int64_t tp = static_cast<int64_t>(k.nch) * L;
  const int nt0 = NT >= NW ? wave : wave % NT, tt0 = NT >= NW ? 0 : wave / NT * LTW;

  f32x4 db[NTW][LTW], dc[NTW][LTW];
#pragma unroll
  for (int j = 0; j < NTW; ++j)
#pragma unroll
    for (int t = 0; t < LTW; ++t) db[j][t] = dc[j][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (t0 < len) {
    {
      Stage<IO, E, NP, L, MNT, VEC> sb, sc;
      sb.init(static_cast<const IO*>(a.bm) + b * a.b_b + static_cast<int64_t>(grp) * a.N, a.b_t, a.N);
      sc.init(static_cast<const IO*>(a.cm) + b * a.c_b + static_cast<int64_t>(grp) * a.N, a.c_t, a.N);
      sb.fetch(t0, len);
      sc.fetch(t0, len);
      sb.commit(Bs);
      sc.commit(Cs);
      for (int i = tid; i < TERM * QE; i += MNT) Qs[i] = Ms[i] = static_cast<E>(0.f);
    }
    Stage<IO, E, PB, L, MNT, VEC> sx, sy;
    float rd, rD;
    float2 rc, rl;
    f32x4 s0[NTW][4], g1[NTW][4];
    const int units = (h1 - h0) * k.pblocks;
    auto fetch = [&](int u) {
      const int h = h0 + u / k.pblocks, p0 = u % k.pblocks * PB;
      sx.init(static_cast<const IO*>(a.x) + b * a.x_b + static_cast<int64_t>(h) * a.P + p0, a.x_t, a.P - p0);
      sy.init(static_cast<const IO*>(k.dy) + b * k.y_b + static_cast<int64_t>(h) * a.P + p0, k.y_t, a.P - p0);
      sx.fetch(t0, len);
      sy.fetch(t0, len);
      const int64_t o = (static_cast<int64_t>(b) * a.H + h) * tp + t0;  // every lane, so that no value is merged
      rd = k.d[o + tid % L];
      rc = k.c[o + tid % L];
      rl = k.c[o + L - 1];
      rD = k.Dz[h];
    };
    auto fetch_states = [&](int u) {
      const int64_t bhp = (static_cast<int64_t>(b) * a.H + h0) * k.pblocks + u;
      const int64_t o = (bhp * k.nch + c) * (NP * PB) + lane * 4;
#pragma unroll
      for (int j = 0; j < NTW; ++j)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int64_t q = o + ((nt0 + NW * j) * 4 + w) * 256;
          s0[j][w] = *reinterpret_cast<const f32x4*>(k.s0 + q);
          g1[j][w] = *reinterpret_cast<const f32x4*>(k.g1 + q);
        }
    };
    auto x_frag = [&](const E* tile, int row0, int k0) {
      if constexpr (XROWS) return packed_frag<E, PB, L>(tile, row0, k0, l16, g);
      else return row_frag<E, PB>(tile, row0, k0, l16, g);
    };
    auto commit = [&](int u) {
      if constexpr (XROWS) sx.commit_rows(Xb[u & 1]);
      else sx.commit(Xb[u & 1]);
      sy.commit(Yb[u & 1]);
      if (tid < L) {
        if (tid == 0) dh2[u & 1] = rD;
        cb2[u & 1][tid] = rc;
        db2[u & 1][tid] = rd;
        eb2[u & 1][tid] = __expf(rc.x + rc.y);
        wb2[u & 1][tid] = decay(rl, rc);
      }
    };
    fetch(0);
    fetch_states(0);
    commit(0);
    fetch(units > 1 ? 1 : 0);
    lds_barrier();
    f32x4 cb[PER];  // C . B of this wave's tiles, transposed (rows s, column t)
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      int tt, st;
      cb[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (!lower_tile<LT>(wave + NW * i, tt, st)) continue;
#pragma unroll
      for (int kb = 0; kb < KN; ++kb)
        cb[i] = mma(row_frag<E, NP>(Bs, 16 * st, 32 * kb, l16, g), row_frag<E, NP>(Cs, 16 * tt, 32 * kb, l16, g), cb[i]);
    }
    for (int u = 0; u < units; ++u) {
      const int h = h0 + u / k.pblocks, pb = u % k.pblocks, p0 = pb * PB;
      const E *Xs = Xb[u & 1], *Ys = Yb[u & 1];
      const float2* cs = cb2[u & 1];
      const float *ds = db2[u & 1], *es = eb2[u & 1], *ws = wb2[u & 1];
      if (u > 0) lds_barrier();  // the last unit's readers of Q, M and G_L are done; this one's inputs are there
      const float Dh = k.has_d ? dh2[u & 1] : 0.f;
      // Q, M and the sums of R
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        int tt, st;
        if (!lower_tile<LT>(wave + NW * i, tt, st)) continue;
        f32x4 xy = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < KP; ++kb)
          xy = mma(x_frag(Xs, 16 * st, 32 * kb), row_frag<E, PB>(Ys, 16 * tt, 32 * kb, l16, g), xy);
        const int t = 16 * tt + l16, s0_ = 16 * st + 4 * g;
        const float2 ct = cs[t];
        const f32x4 c01 = *reinterpret_cast<const f32x4*>(cs + s0_), c23 = *reinterpret_cast<const f32x4*>(cs + s0_ + 2);
        const f32x4 dv = *reinterpret_cast<const f32x4*>(ds + s0_);
        struct alignas(4 * sizeof(E)) M4 { E e[4]; } q[TERM], m[TERM];
        float dg = 0.f, rr[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool on = s0_ + r <= t;
          const float2 from = make_float2((r < 2 ? c01 : c23)[2 * (r & 1)], (r < 2 ? c01 : c23)[2 * (r & 1) + 1]);
          const float w = decay(ct, from), wd = w * dv[r];
          float xq = xy[r] * wd, cm_ = cb[i][r] * wd;
          const float xc = cb[i][r] * xy[r] * w;  // off the triangle: dropped, not added
          xq = on ? xq : 0.f, cm_ = on ? cm_ : 0.f;
#pragma unroll
          for (int k = 0; k < TERM; ++k) {
            q[k].e[r] = static_cast<E>(xq), m[k].e[r] = static_cast<E>(cm_);
            xq -= static_cast<float>(q[k].e[r]), cm_ -= static_cast<float>(m[k].e[r]);
          }
          rr[r] = on ? xc : 0.f;
          dg = s0_ + r == t ? xy[r] : dg;
        }
        const int o = TQ::at(t) + 16 * st + 4 * g;
#pragma unroll
        for (int k = 0; k < TERM; ++k) {
          *reinterpret_cast<M4*>(Qs + k * QE + o) = q[k];
          *reinterpret_cast<M4*>(Ms + k * QE + o) = m[k];
        }
        // left of the diagonal the rows' sums, in a tile on it each token's sum over the paths that cross it
        float rs = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float from_t = row16_suffix(rr[r]);  // sum over the tokens from t on
          const float v = tt != st ? rr[r] : s0_ + r < t ? from_t : 0.f;
          rs = fmaf(v, dv[r], rs);
          rr[r] = from_t;
        }
        rs = half_pair_sum(row_pair_sum(rs));
        if (g == 0) row_r[st][t] = rs;
        if (l16 == 0) *reinterpret_cast<float4*>(&col_r[tt][16 * st + 4 * g]) = make_float4(rr[0], rr[1], rr[2], rr[3]);
        if (tt == st) {
          dg = half_pair_sum(row_pair_sum(row16_sum(dg)));
          if (lane == 0) diag[tt] = dg;
        }
      }
      // S_0^T dy and G_L^T x (rows n, column t or s)
      float kp = 0.f, al[LTW] = {}, be[LTW] = {};
#pragma unroll
      for (int j = 0; j < NTW; ++j) {
        const int n = 16 * (nt0 + NW * j) + 4 * g;
#pragma unroll
        for (int kb = 0; kb < KP; ++kb)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int r = 0; r < 4; ++r) kp = fmaf(s0[j][2 * kb + hf][r], g1[j][2 * kb + hf][r], kp);
#pragma unroll
        for (int which = 0; which < 2; ++which) {  // one after the other: the registers of one
          f32x4 prod[LTW];
#pragma unroll
          for (int t = 0; t < LTW; ++t) prod[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kb = 0; kb < KP; ++kb) {
            Frag<E> part[NPART], f[LTW];
#pragma unroll
            for (int t = 0; t < LTW; ++t)
              f[t] = which ? x_frag(Xs, 16 * (tt0 + t), 32 * kb) : row_frag<E, PB>(Ys, 16 * (tt0 + t), 32 * kb, l16, g);
            const f32x4 v[2] = {which ? g1[j][2 * kb] : s0[j][2 * kb], which ? g1[j][2 * kb + 1] : s0[j][2 * kb + 1]};
            split<E>(v, part);
#pragma unroll
            for (int q = NPART - 1; q >= 0; --q)
#pragma unroll
              for (int t = 0; t < LTW; ++t) prod[t] = mma(part[q], f[t], prod[t]);
          }
#pragma unroll
          for (int t = 0; t < LTW; ++t) {
            const int tok = 16 * (tt0 + t) + l16;
            const E* row = (which ? Bs : Cs) + TB::at(tok) + n;
            const float w = which ? ws[tok] : es[tok], d = which ? ds[tok] : 1.f;
            f32x4& sum = which ? db[j][t] : dc[j][t];
            float& dot = which ? be[t] : al[t];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float v = prod[t][r] * w;
              dot = fmaf(static_cast<float>(row[r]), v, dot);
              sum[r] = fmaf(d, v, sum[r]);
            }
          }
        }
      }
      f32x4 dx[2];
      const int pt = wave & 3, st0 = (wave >> 2) * (LT / 2);  // dx: p-tile, s-tiles st0 .. st0 + LT / 2 - 1
      constexpr int DXT = LT / 2;
#pragma unroll
      for (int t = 0; t < DXT; ++t) dx[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int hh = 0; hh < NH; ++hh) {
        if (hh > 0) lds_barrier();
#pragma unroll
        for (int j = 0; j < NTW; ++j) {
          const int tile = nt0 + NW * j;
          if (tile / (GR / 16) != hh || (NT < NW && tt0 != 0)) continue;
#pragma unroll
          for (int w = 0; w < 4; w += 2) {
            f32x4 v[2] = {g1[j][w], g1[j][w + 1]};
            asm volatile("" : "+v"(v[0]), "+v"(v[1]));  // rounded again: the products' parts held until here would spill
            Frag<E> part[TERM];
            split<E, TERM, true>(v, part);
#pragma unroll
            for (int k = 0; k < TERM; ++k) {
              E* o = Gs + k * GE + TX::at(16 * (tile % (GR / 16)) + l16) + 16 * w + 4 * g;
              put_half(o, part[k], 0);
              put_half(o + 16, part[k], 1);
            }
          }
        }
        if (hh == 0) {
#pragma unroll
          for (int t = 0; t < LTW; ++t) {
            const float v = half_pair_sum(row_pair_sum(al[t])), w = half_pair_sum(row_pair_sum(be[t]));
            if (g == 0) alpha[nt0][16 * (tt0 + t) + l16] = v, beta[nt0][16 * (tt0 + t) + l16] = w;
          }
          kp = half_pair_sum(row_pair_sum(row16_sum(kp)));
          if (lane == 0) kappa[wave] = NT >= NW || tt0 == 0 ? kp : 0.f;
        }
        if (hh == NH - 1) fetch_states(u + 1 < units ? u + 1 : u);
        lds_barrier();
        if (hh == NH - 1 && u + 1 < units) {  // into the other buffers: the unit before this one is done with them
          commit(u + 1);
          fetch(u + 2 < units ? u + 2 : u + 1);  // always, and the states too: a load under a condition is waited for where its value merges
        }
#pragma unroll
        for (int kb = 0; kb < GR / 32; ++kb) {
          Frag<E> gf[TERM], bf[DXT];
#pragma unroll
          for (int i = 0; i < TERM; ++i) gf[i] = col_frag<E, PB>(Gs + i * GE, 32 * kb, 16 * pt, l16, g);
#pragma unroll
          for (int t = 0; t < DXT; ++t) bf[t] = row_frag<E, NP>(Bs, 16 * (st0 + t), GR * hh + 32 * kb, l16, g);
#pragma unroll
          for (int i = TERM - 1; i >= 0; --i)
#pragma unroll
            for (int t = 0; t < DXT; ++t) dx[t] = mma(gf[i], bf[t], dx[t]);
        }
      }
      // the chunk's own terms
#pragma unroll
      for (int j = 0; j < NTW; ++j) {
#pragma unroll
        for (int kb = 0; kb < KL; ++kb) {
          const Frag<E> bf = col_frag<E, NP>(Bs, 32 * kb, 16 * (nt0 + NW * j), l16, g);
          const Frag<E> cf = col_frag<E, NP>(Cs, 32 * kb, 16 * (nt0 + NW * j), l16, g);
#pragma unroll
          for (int i = TERM - 1; i >= 0; --i)
#pragma unroll
            for (int t = 0; t < LTW; ++t) {
              if ((tt0 + t) / 2 >= kb) dc[j][t] = mma(bf, row_frag<E, L>(Qs + i * QE, 16 * (tt0 + t), 32 * kb, l16, g), dc[j][t]);
              if ((tt0 + t) / 2 <= kb) db[j][t] = mma(cf, col_frag<E, L>(Qs + i * QE, 32 * kb, 16 * (tt0 + t), l16, g), db[j][t]);
            }
        }
      }
#pragma unroll
      for (int t = 0; t < DXT; ++t) {
        const int st = st0 + t, s = 16 * st + l16;
        dx[t] *= ws[s] * ds[s];
#pragma unroll
        for (int kb = 0; kb < KL; ++kb) {
          if (st / 2 > kb) continue;
          const Frag<E> yf = col_frag<E, PB>(Ys, 32 * kb, 16 * pt, l16, g);
#pragma unroll
          for (int i = TERM - 1; i >= 0; --i) dx[t] = mma(yf, col_frag<E, L>(Ms + i * QE, 32 * kb, 16 * st, l16, g), dx[t]);
        }
        const int p = p0 + 16 * pt + 4 * g;
        if (t0 + s < a.T && p < a.P && k.dx != nullptr) {
          const E* yr = Ys + TX::at(s) + 16 * pt + 4 * g;
          // a scalar base and a lane's offset
          IO* o = static_cast<IO*>(k.dx) + ((static_cast<int64_t>(b) * a.T + t0) * a.H + h) * a.P + p0 + (s * a.H * a.P + 16 * pt + 4 * g);
          f32x4 q;
#pragma unroll
          for (int r = 0; r < 4; ++r) q[r] = fmaf(Dh, static_cast<float>(yr[r]), dx[t][r]);
          if (t0 + L > len) {  // behind the length 0, whatever a NaN made of the zeros there
#pragma unroll
            for (int r = 0; r < 4; ++r) q[r] = t0 + s < len ? q[r] : 0.f;
          }
          const Out4<IO> v = out4<IO>(q);
          if (k.vec_dx) {
            *reinterpret_cast<Out4<IO>*>(o) = v;
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (p + r < a.P) o[r] = v.e[r];
          }
        }
      }
      // what the step sizes' gradients are made of, for steps_kernel: the last four waves a sum each
      {
        const int64_t bhp = (static_cast<int64_t>(b) * a.H + h) * k.pblocks + pb, plane = static_cast<int64_t>(a.B) * a.H * k.pblocks;
        const int which = wave - (NW - 4), t = lane % L;
        if (which >= 0) {
          constexpr int NS = NT < NW ? NT : NW;
          float v = 0.f;
          if (which == 2) {
            const int tile = t / 16;
            float row = 0.f, col = 0.f;
#pragma unroll
            for (int i = 0; i < LT; ++i) {
              row += i < tile ? row_r[i][t] : 0.f;
              col += i > tile ? col_r[i][t] : 0.f;
            }
            col *= ds[t];
            v = row_r[tile][t] + row16_suffix(row) + row16_before(col);
#pragma unroll
            for (int m = 1; m < LT - 1; ++m) {  // the tiles wholly across tile m
              float over = 0.f;
#pragma unroll
              for (int i = 0; i < m; ++i) over += tile > m ? row_r[i][t] : 0.f;
              over = half_pair_sum(row_pair_sum(row16_sum(over)));
              v += tile == m ? over : 0.f;
            }
          } else if (which < 2) {
#pragma unroll
            for (int i = 0; i < NS; ++i) v += which == 0 ? alpha[i][t] : beta[i][t];
          } else {
#pragma unroll
            for (int i = 0; i < LT; ++i) {  // (slots of tiles right of the diagonal hold nothing)
              const float w = col_r[i][t];
              v += i >= t / 16 ? w : 0.f;
            }
          }
          if (lane < L) k.tok[(which * plane + bhp) * tp + t0 + t] = v;
          if (lane == 0 && which < 2) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < NW; ++i) s += which == 0 ? kappa[i] : i < LT ? diag[i] : 0.f;
            k.chk[(which * plane + bhp) * k.nch + c] = which == 0 ? s * es[L - 1] : s;
          }
        }
      }
    }
  } else {  // behind the sequence's end
    for (int h = h0; h < h1; ++h) {
      const int rows = min(L, a.T - t0);
      if (k.dx != nullptr)
        for (int t = wave; t < rows; t += NW)
          for (int p = lane; p < a.P; p += 64)
            io<IO>::store(static_cast<IO*>(k.dx) + ((static_cast<int64_t>(b) * a.T + t0 + t) * a.H + h) * a.P, p, 0.f);
    }
  }
  // dB, dC: rows n, column t
#pragma unroll
  for (int j = 0; j < NTW; ++j) {
    const int n = 16 * (nt0 + NW * j) + 4 * g;
#pragma unroll
    for (int t = 0; t < LTW; ++t) {
      const int tok = t0 + 16 * (tt0 + t) + l16;
      if (tok >= a.T || n >= a.N) continue;
      if (tok >= len) db[j][t] = dc[j][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int64_t o = ((static_cast<int64_t>(b) * a.T + tok) * a.G + grp) * a.N + n;
      const int64_t part = static_cast<int64_t>(hb) * a.B * a.T * a.G * a.N;
      if (k.pb != nullptr && a.N % 4 == 0) {
        *reinterpret_cast<f32x4*>(k.pb + part + o) = db[j][t];
        *reinterpret_cast<f32x4*>(k.pc + part + o) = dc[j][t];
        continue;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (n + r >= a.N) continue;
        if (k.pb != nullptr) {
          k.pb[part + o + r] = db[j][t][r];
          k.pc[part + o + r] = dc[j][t][r];
        } else {
          if (k.db != nullptr) io<IO>::store(static_cast<IO*>(k.db), o + r, db[j][t][r]);
          if (k.dc != nullptr) io<IO>::store(static_cast<IO*>(k.dc), o + r, dc[j][t][r]);
        }
      }
    }
  }
}

// The gradients of a chunk's step sizes, a lane a token.
template <int L>
__global__ __launch_bounds__(SNT) void steps_kernel(Bwd k, int64_t units) {
  const Args& a = k.a;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (SNT / 64) + (threadIdx.x >> 6);
  if (unit >= units) return;
  const int lane = threadIdx.x & 63;
  const int h = static_cast<int>(unit % a.H);
  const int64_t bc = unit / a.H;
  const int b = static_cast<int>(bc / k.nch), c = static_cast<int>(bc - static_cast<int64_t>(b) * k.nch);
  const int len = length_of(a.lengths, a.lengths64, a.T, b), t = c * L + lane;
  const int64_t bh = static_cast<int64_t>(b) * a.H + h, tp = static_cast<int64_t>(k.nch) * L;
  const int64_t plane = static_cast<int64_t>(a.B) * a.H * k.pblocks;
  const bool in = lane < L && t < len;
  double dz = 0.0, ga = 0.0, dgs = 0.0;
  if (c * L < len) {
    double al = 0.0, be = 0.0, in_g = 0.0, cr = 0.0, kap = 0.0, d = 0.0;
    for (int p = 0; p < k.pblocks; ++p) {
      const int64_t row = bh * k.pblocks + p;
      kap += k.chk[row * k.nch + c];
      dgs += k.chk[(plane + row) * k.nch + c];
      const float* tok = k.tok + row * tp + c * L + lane % L;
      const float v[4] = {tok[0], tok[plane * tp], tok[2 * plane * tp], tok[3 * plane * tp]};
      al += in ? v[0] : 0.f;
      be += in ? v[1] : 0.f;
      in_g += in ? v[2] : 0.f;
      cr += in ? v[3] : 0.f;
    }
    const float dt = k.d[bh * tp + c * L + lane % L];
    d = in ? dt : 0.f;
    double suf = al, pre = d * be;
    const double own = pre;
#pragma unroll
    for (int off = 1; off < L; off <<= 1) {
      const double v = __shfl_down(suf, off, 64), w = __shfl_up(pre, off, 64);
      if (lane + off < L) suf += v;
      if (lane >= off) pre += w;
    }
    const double gt = kap + in_g + suf + (pre - own);
    // sigmoid(z) = 1 - e^{-softplus(z)}
    const double slope = a.softplus ? static_cast<double>(-expm1f(-static_cast<float>(d))) : 1.0;
    if (in) {
      dz = (cr + be + static_cast<double>(a.A[h]) * gt) * slope;
      ga = d * gt;
    }
  }
  if (lane < L && t < a.T && k.ddelta != nullptr) {
    const int64_t o = (static_cast<int64_t>(b) * a.T + t) * a.H + h;
    const float v = static_cast<float>(dz);
    if (a.delta_dtype == VMI_F32) io<float>::store(static_cast<float*>(k.ddelta), o, v);
    else if (a.delta_dtype == VMI_BF16) io<bf16_t>::store(static_cast<bf16_t*>(k.ddelta), o, v);
    else io<f16_t>::store(static_cast<f16_t*>(k.ddelta), o, v);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) dz += __shfl_xor(dz, off), ga += __shfl_xor(ga, off);
  if (lane != 0) return;
  const int64_t rows = static_cast<int64_t>(a.B) * k.nch, o = bc * a.H + h;
  k.ph[o] = static_cast<float>(ga);
  k.ph[rows * a.H + o] = static_cast<float>(dgs);
  k.ph[2 * rows * a.H + o] = static_cast<float>(dz);
}

// Blocks below `heads`: 16 of the 3 H head sums by 16 strided shares of the chunks.  The others: dB and dC
// from the head blocks' partials.
template <typename IO>
__global__ __launch_bounds__(SNT) void reduce_kernel(Bwd k, int heads, int64_t elems) {
  const Args& a = k.a;
  if (static_cast<int>(blockIdx.x) < heads) {
    constexpr int COLS = 16, SHARES = SNT / COLS;
    __shared__ double part[SHARES][COLS];
    const int l = threadIdx.x % COLS, share = threadIdx.x / COLS, col = blockIdx.x * COLS + l;
    const int64_t rows = static_cast<int64_t>(a.B) * k.nch;
    double s = 0.0;
    const int which = col / a.H, h = col - which * a.H;
    if (which < 3)
      for (int64_t r = share; r < rows; r += SHARES) s += k.ph[(which * rows + r) * a.H + h];
    part[share][l] = s;
    __syncthreads();
    if (share != 0 || which >= 3) return;
    float* dst = which == 0 ? k.dA : which == 1 ? k.dD : k.dbias;
    for (int i = 1; i < SHARES; ++i) s += part[i][l];
    if (dst != nullptr) dst[h] = static_cast<float>(s);
    return;
  }
  const int64_t i = (static_cast<int64_t>(blockIdx.x - heads) * SNT + threadIdx.x) * 4;
  if (i >= elems) return;
  const int left = static_cast<int>(elems - i < 4 ? elems - i : 4);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const float* part = which ? k.pc : k.pb;
    IO* dst = static_cast<IO*>(which ? k.dc : k.db);
    if (dst == nullptr) continue;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (elems % 4 == 0) {
      for (int q = 0; q < k.hblocks; ++q) v += *reinterpret_cast<const f32x4*>(part + q * elems + i);
      if (reinterpret_cast<uintptr_t>(dst) % (4 * sizeof(IO)) == 0) {
        *reinterpret_cast<Out4<IO>*>(dst + i) = out4<IO>(v);
        continue;
      }
    } else {
      for (int q = 0; q < k.hblocks; ++q)
        for (int r = 0; r < left; ++r) v[r] += part[q * elems + i + r];
    }
    for (int r = 0; r < left; ++r) io<IO>::store(dst, i + r, v[r]);
  }
}

namespace {

int bwd_tokens(int dtype, int64_t N) { return dtype == VMI_BF16 && N <= 128 ? 64 : 32; }

struct Plan {
  int64_t nch, tp, c_bytes, d_bytes, own_bytes, state_bytes, part_bytes, ph_bytes, tok_bytes, chk_bytes;
  int np, pblocks, seg_chunks, nseg, hblocks, hper;
  int64_t bytes() const { return c_bytes + d_bytes + own_bytes + 2 * state_bytes + 2 * part_bytes + ph_bytes + tok_bytes + chk_bytes; }
};

Plan plan(int64_t B, int64_t T, int64_t H, int64_t P, int64_t G, int64_t N, int dtype) {
  Plan p;
  const int L = bwd_tokens(dtype, N);
  p.np = N <= 64 ? 64 : N <= 128 ? 128 : 256;
  p.nch = (T + L - 1) / L;
  p.tp = p.nch * L;
  p.pblocks = static_cast<int>((P + PB - 1) / PB);
  const int64_t BHP = B * H * p.pblocks, want = (256 + 2 * BHP - 1) / (2 * BHP);
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(BWD_MAX_SEG, p.nch / 4));
  const int64_t nseg = std::min(want, most);
  p.seg_chunks = static_cast<int>((p.nch + nseg - 1) / nseg);
  p.nseg = static_cast<int>((p.nch + p.seg_chunks - 1) / p.seg_chunks);
  const int64_t hg = H / G, blocks = B * p.nch * G, split = std::min<int64_t>(hg, (256 + blocks - 1) / blocks);
  p.hper = static_cast<int>((hg + split - 1) / split);
  p.hblocks = static_cast<int>((hg + p.hper - 1) / p.hper);
  p.c_bytes = up16(B * H * p.tp * 8);
  p.d_bytes = up16(B * H * p.tp * 4);
  const int64_t state = static_cast<int64_t>(p.np) * PB * 4;
  p.own_bytes = p.nseg > 1 ? 2 * p.nseg * BHP * state : 0;
  p.state_bytes = BHP * p.nch * state;
  p.part_bytes = p.hblocks > 1 ? up16(p.hblocks * B * T * G * N * 4) : 0;
  p.ph_bytes = up16(3 * B * p.nch * H * 4);
  p.tok_bytes = up16(4 * BHP * p.tp * 4);
  p.chk_bytes = up16(2 * BHP * p.nch * 4);
  return p;
}

template <typename IO, typename E, int NP, int L, bool VEC> int run(Bwd k, const Plan& p, hipStream_t stream) {
  const Args& a = k.a;
  const int64_t BHP = static_cast<int64_t>(a.B) * a.H * p.pblocks, wgs = BHP * p.nseg;
  const int64_t blocks = static_cast<int64_t>(a.B) * p.nch * a.G * p.hblocks;
  if (!grid_fits(wgs, SNT) || !grid_fits(blocks, MNT)) return VMI_ERR_UNSUPPORTED;
  auto ok = [](int& st) { return (st = hip_status(hipGetLastError())) == VMI_OK; };
  int st = launch_prep(a, L, const_cast<float*>(k.d), const_cast<float2*>(k.c), static_cast<int>(p.nch), stream);
  if (st != VMI_OK) return st;
  const dim3 grid(static_cast<unsigned>(wgs), 2);
  if (p.nseg > 1) {
    hipLaunchKernelGGL((states_kernel<IO, E, NP, L, true, VEC>), grid, dim3(SNT), 0, stream, k);
    if (!ok(st)) return st;
    const int64_t pieces = (BHP * (NP * PB / 4) + SNT - 1) / SNT;
    if (!grid_fits(pieces, SNT)) return VMI_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(starts_kernel<NP>, dim3(static_cast<unsigned>(pieces), 2), dim3(SNT), 0, stream, k, L);
    if (!ok(st)) return st;
  }
  hipLaunchKernelGGL((states_kernel<IO, E, NP, L, false, VEC>), grid, dim3(SNT), 0, stream, k);
  if (!ok(st)) return st;
  hipLaunchKernelGGL((main_kernel<IO, E, NP, L, VEC>), dim3(static_cast<unsigned>(blocks)), dim3(MNT), 0, stream, k);
  if (!ok(st)) return st;
  const int64_t chunks = static_cast<int64_t>(a.B) * a.H * p.nch, sb = (chunks + SNT / 64 - 1) / (SNT / 64);
  if (!grid_fits(sb, SNT)) return VMI_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(steps_kernel<L>, dim3(static_cast<unsigned>(sb)), dim3(SNT), 0, stream, k, chunks);
  if (!ok(st)) return st;
  const int heads = (3 * a.H + 15) / 16;
  const int64_t elems = static_cast<int64_t>(a.B) * a.T * a.G * a.N;
  const int64_t rb = heads + (p.hblocks > 1 ? (elems + 4 * SNT - 1) / (4 * SNT) : 0);
  if (!grid_fits(rb, SNT)) return VMI_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(reduce_kernel<IO>, dim3(static_cast<unsigned>(rb)), dim3(SNT), 0, stream, k, heads, elems);
  ok(st);
  return st;
}

// Chunks of MOST tokens up to 128 state columns, of 32 above.
template <typename IO, typename E, int MOST> int by_state(const Bwd& k, const Plan& p, hipStream_t stream) {
  auto go = [&](auto np) -> int {
    constexpr int NP = decltype(np)::value, L = NP > 128 ? 32 : MOST;
    return k.vec ? run<IO, E, NP, L, true>(k, p, stream) : run<IO, E, NP, L, false>(k, p, stream);
  };
  if (p.np == 64) return go(std::integral_constant<int, 64>{});
  if (p.np == 128) return go(std::integral_constant<int, 128>{});
  return go(std::integral_constant<int, 256>{});
}

}  // namespace

size_t bwd_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t P, int64_t G, int64_t N, int dtype) {
  return static_cast<size_t>(plan(B, T, H, P, G, N, dtype).bytes());
}

int launch_bwd(const Args& a, int dtype, const Grads& q, void* workspace, hipStream_t stream) {
  const Plan p = plan(a.B, a.T, a.H, a.P, a.G, a.N, dtype);
  Bwd k{};
  k.a = a;
  k.dy = q.dy, k.y_t = q.y_t, k.y_b = q.y_b, k.dstate = q.dstate;
  k.dx = q.dx, k.ddelta = q.ddelta, k.db = q.db, k.dc = q.dc, k.dA = q.dA, k.dD = q.dD, k.dbias = q.dbias;
  k.dstate_in = q.dstate_in;
  k.has_d = a.D != nullptr, k.Dz = k.has_d ? a.D : a.A;
  char* w = static_cast<char*>(workspace);
  auto take = [&](int64_t bytes) {
    char* r = w;
    w += bytes;
    return r;
  };
  k.c = reinterpret_cast<const float2*>(take(p.c_bytes));
  k.d = reinterpret_cast<const float*>(take(p.d_bytes));
  k.own = reinterpret_cast<float*>(take(p.own_bytes));
  k.s0 = reinterpret_cast<float*>(take(p.state_bytes));
  k.g1 = reinterpret_cast<float*>(take(p.state_bytes));
  if (p.hblocks > 1) {
    k.pb = reinterpret_cast<float*>(take(p.part_bytes));
    k.pc = reinterpret_cast<float*>(take(p.part_bytes));
  }
  k.ph = reinterpret_cast<float*>(take(p.ph_bytes));
  k.tok = reinterpret_cast<float*>(take(p.tok_bytes));
  k.chk = reinterpret_cast<float*>(take(p.chk_bytes));
  k.nch = static_cast<int>(p.nch), k.seg_chunks = p.seg_chunks, k.nseg = p.nseg, k.pblocks = p.pblocks;
  k.hblocks = p.hblocks, k.hper = p.hper;
  const int el = dtype == VMI_F32 ? 4 : 8;
  k.vec = a.P % el == 0 && a.x_t % el == 0 && a.x_b % el == 0 && q.y_t % el == 0 && q.y_b % el == 0 &&
          a.N % el == 0 && a.b_t % el == 0 && a.b_b % el == 0 && a.c_t % el == 0 && a.c_b % el == 0 &&
          aligned16({a.x, q.dy, a.bm, a.cm});
  k.vec_dx = a.P % 4 == 0 && aligned16({q.dx});
  if (dtype == VMI_BF16) return by_state<bf16_t, __bf16, 64>(k, p, stream);
  if (dtype == VMI_F16) return by_state<f16_t, float, 32>(k, p, stream);
  return by_state<float, float, 32>(k, p, stream);
}

}  // namespace sel
}  // namespace vmi
