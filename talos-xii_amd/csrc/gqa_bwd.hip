// gqa_bwd.hip -- grouped-query attention, backward: the probabilities formed again from the forward's lse.
//
//   p_ij = exp2(c s_ij + b_ij - lse2_i),   D_i = sum_d dO_id O_id,   dS_ij = p_ij (dO_i . v_j - D_i)
//   dQ_i = scale sum_j dS_ij k_j,   dV_j = sum_i p_ij dO_i,   dK_j = scale sum_i dS_ij q_i,   dbias = sums of dS by j - i
//
// Two kernels, each owning what it sums, so nothing is added atomically and every sum has one order:
// * dQ (and D): a wave holds 32 rows of a group (as in the forward) and walks the keys: S^T = K Q^T, dP^T = V dO^T,
//   dQ^T += K^T dS^T, with dS^T straight from the accumulator.
// * dK and dV: a wave holds 32 keys and walks the queries of the group's heads, one head after the other:
//   S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS. The heads of a group add into the same registers.
// That is seven block products where one kernel that adds dQ atomically would need five.
//
// D of a bf16 o. The forward's o carries the rounding of its probabilities and its own, 2^-9 of o each, and D from it is
// off by that share of dO o: nothing beside dS's own rounding in rows that look at many keys, but of a row that sees few o
// is as large as v (18 ragged tokens: error of dQ 3.1e-3 for 2.3e-3), and in dbias the error of a row meets the same
// distances again and again (2.7e-3 of dbias at 2 x 2048 tokens, where its fp32 sums are good to 1e-6). But sum_j dS_ij = 0
// says what is missing: with D' from o, R_i = sum_j p_ij (dP_ij - D'_i) is D - D', formed in fp32 beside the rest. The
// dK / dV kernel, which runs after the dQ kernel, gets D' + R. dQ needs R times sum_j p_ij k_j as well, one more block
// product, whose accumulators spill at d 128 (216 registers without it): workgroups of rows that see few keys run a kernel
// with it, the others one without (4 x 4096 tokens, d 128, forward and backward 1459 us; all with it 1580).
//
// The bias gradient belongs to the second kernel, where one head is at work: a block of 32 keys by 32 queries spans 63
// distances. Blocks at least M away add into one register a lane; nearer ones sum their diagonals in registers
// (diagonals() below) and add them, one lane a distance, to an array by distance in LDS that is the wave's own: no two
// additions meet, and the order is the program's. The four arrays are folded once a head. (Sixteen LDS float atomics a
// block, each lane its values, cost 224 cycles apiece: 127 us of 322 at 2 x 2048 tokens, 16 heads, d 64, M 128.)
#include <algorithm>
#include <climits>
#include <type_traits>

#include "gqa.hpp"

namespace talos {

namespace {

template <typename T, int D, int NK, int NBUF>
struct DqShape {
  static constexpr int NP = kPlanes<T>, ROWS = 128, BUF = 2 * NP * NK * D;
  static constexpr size_t lds = (size_t)NBUF * BUF * 2;
};

// waves a SIMD that the kernels are compiled for, as in the forward (which has the figures)
template <typename T, int D, bool DMA>
constexpr int kBwdWaves = D == 128 && !DMA ? 1 : 2;

// BIAS, DMA: as in the forward. FIX (bf16): dQ is corrected by R, for the workgroups whose rows see at most a.few keys; the
// others are the kernel's without it.
template <typename T, int D, int NK, int NBUF, bool BIAS, bool DMA, bool FIX>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kBwdWaves<T, D, DMA>))) void gqa_dq_kernel(GqaArgs a) {
  constexpr bool REST = sizeof(T) == 2;  // R is summed
  static_assert(REST || !FIX, "fp32 rows have an exact D");
  using S = DqShape<T, D, NK, NBUF>;
  constexpr int NP = S::NP, KS = D / 16, OB = D / 32, KB = NK / 32, PL = NK * D;
  extern __shared__ __align__(16) uint16_t lds[];
  const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5, wv = gq_wave();
  const GqaItem it = gq_item(a, true);
  const GqaSample sm = gq_sample(a, it.b);
  const int G = a.G;
  const int row0 = it.tile * S::ROWS + wv * 32, row = row0 + l32;
  const int qi = row / G, head = it.kvh * G + row % G;
  const bool live = qi < sm.ql;
  const int lim = !live ? 0 : a.causal ? min(sm.kl, qi + sm.off + 1) : sm.kl;
  const int q_lo = row0 / G, q_hi = min((row0 + 31) / G, sm.ql - 1);
  const int lim_lo = a.causal ? min(sm.kl, q_lo + sm.off + 1) : sm.kl;
  const int lim_hi = q_lo >= sm.ql ? 0 : a.causal ? min(sm.kl, q_hi + sm.off + 1) : sm.kl;
  const int wg_lo = it.tile * S::ROWS / G, wg_hi = min((it.tile * S::ROWS + S::ROWS - 1) / G, sm.ql - 1);
  const int kend = wg_lo >= sm.ql ? 0 : a.causal ? max(0, min(sm.kl, wg_hi + sm.off + 1)) : sm.kl;
  if (REST && FIX != (kend <= a.few)) return;
  const int ntile = (kend + NK - 1) / NK;
  const int t_beg = (int)((long long)ntile * it.split / a.splits), t_end = (int)((long long)ntile * (it.split + 1) / a.splits);

  const T* kbase = static_cast<const T*>(a.k) + (long long)it.b * a.Sk * a.ldk + (long long)it.kvh * a.dk;
  const T* vbase = static_cast<const T*>(a.v) + (long long)it.b * a.Sk * a.ldv + (long long)it.kvh * a.dv;
  std::conditional_t<DMA, GqaDma<D, NK>, GqaTile<T, D, NK>> kt, vt;
  if constexpr (DMA) {
    kt.init(a.ldk);
    vt.init(a.ldv);
  }
  if (t_beg < t_end) {
    if constexpr (DMA) {
      uint16_t* buf = lds + (t_beg & 1) * S::BUF;
      kt.issue(kbase, a.ldk, t_beg * NK, sm.kl, buf);
      vt.issue(vbase, a.ldv, t_beg * NK, sm.kl, buf + PL);
    } else {
      kt.fetch(kbase, a.ldk, t_beg * NK, sm.kl, a.dk);
      vt.fetch(vbase, a.ldv, t_beg * NK, sm.kl, a.dv);
    }
  }
  Frag<NP> qf[KS], gf[KS];
  float delta = 0.f, lse2 = INFINITY;
  const long long at = ((long long)it.b * a.H + head) * a.Sq + (qi < a.Sq ? qi : 0);
  {
    const long long token = (long long)it.b * a.Sq + (live ? qi : 0);
    const T* qrow = static_cast<const T*>(a.q) + token * a.ldq + (long long)head * a.dk;
    const T* grow = static_cast<const T*>(a.dout) + token * a.lddo + (long long)head * a.dv;
    const T* orow = static_cast<const T*>(a.o) + token * a.ldo + (long long)head * a.dv;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      Eight<T> e, g, o;
      const int c = 16 * s + 8 * h;
      e.zero();
      g.zero();
      o.zero();
      if (live && c < a.dk) e.load(qrow, c, a.dk);
      if (live && c < a.dv) {
        g.load(grow, c, a.dv);
        o.load(orow, c, a.dv);
      }
      delta += g.dot(o);
      qf[s] = gq_frag(e);
      gf[s] = gq_frag(g);
    }
    delta = gq_sum_halves(delta);
    if (live) {
      const float x = a.lse[at];
      lse2 = x == -INFINITY ? INFINITY : x * kLog2e;  // a row that saw no key: p = 0
    }
  }
  const float* bias = nullptr;
  float bias_l = 0.f, bias_r = 0.f;
  const int pos = qi + sm.off;
  if (BIAS) {
    bias = a.bias + (size_t)(live ? head : 0) * (2 * a.M + 1) + a.M;
    bias_l = gq_bias(bias[-a.M]);
    bias_r = gq_bias(bias[a.M]);
  }

  GqaLane<D> ln;
  gq_f32x16 acc[OB], pk[FIX ? OB : 1];
  float rest = 0.f;
#pragma unroll
  for (int i = 0; i < OB; ++i) {
    acc[i] = gq_zero();
    if (FIX) pk[i] = gq_zero();
  }

  for (int t = t_beg; t < t_end; ++t) {
    uint16_t* buf = lds + (NBUF == 2 ? (t & 1) * S::BUF : 0);
    if constexpr (DMA) {
      gq_dma_wait();
      __syncthreads();
      if (t + 1 < t_end) {
        uint16_t* next = lds + ((t + 1) & 1) * S::BUF;
        kt.issue(kbase, a.ldk, (t + 1) * NK, sm.kl, next);
        vt.issue(vbase, a.ldv, (t + 1) * NK, sm.kl, next + PL);
      }
    } else {
      if (NBUF == 1 && t != t_beg) __syncthreads();
      kt.stash(buf);
      vt.stash(buf + NP * PL);
      if (t + 1 < t_end) {
        kt.fetch(kbase, a.ldk, (t + 1) * NK, sm.kl, a.dk);
        vt.fetch(vbase, a.ldv, (t + 1) * NK, sm.kl, a.dv);
      }
      __syncthreads();
    }
    const uint16_t *Kt = buf, *Vt = buf + NP * PL;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int k0 = t * NK + 32 * kb;
      if (k0 >= lim_hi) continue;
      ln.renew();
      gq_f32x16 s = gq_zero(), dp = gq_zero();
      {
        gq_f32x16 lo = gq_zero(), lo2 = gq_zero();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const Frag<NP> kf = gq_frag_row<NP, D, PL>(Kt, ln, kb * 32, ks);
          if constexpr (NP == 3) lo = gq_mfma_small(kf, qf[ks], lo);
          s = gq_mfma(kf.p[0], qf[ks].p[0], s);
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const Frag<NP> vf = gq_frag_row<NP, D, PL>(Vt, ln, kb * 32, ks);
          if constexpr (NP == 3) lo2 = gq_mfma_small(vf, gf[ks], lo2);
          dp = gq_mfma(vf.p[0], gf[ks].p[0], dp);
        }
        if constexpr (NP == 3) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            s[r] += lo[r];
            dp[r] += lo2[r];
          }
        }
      }
      float mul = a.c, sub = -lse2;
      if (BIAS) {
        if (k0 + 31 - (q_lo + sm.off) <= -a.M) {
          sub += bias_l;
        } else if (k0 - (q_hi + sm.off) >= a.M) {
          sub += bias_r;
        } else {
          mul = 1.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int d = k0 + gq_row(r, h) - pos;
            s[r] = fmaf(s[r], a.c, gq_bias(bias[min(max(d, -a.M), a.M)]));
          }
        }
      }
      if (k0 + 32 > lim_lo) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (k0 + gq_row(r, h) >= lim) {
            s[r] = -INFINITY;
            dp[r] = 0.f;
          }
      }
      float p[16], ds[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = __builtin_amdgcn_exp2f(fmaf(s[r], mul, sub));
        ds[r] = p[r] * (dp[r] - delta);
        if (REST) rest += ds[r];
      }
      const Frag<NP> df[2] = {gq_frag_acc<NP>(ds), gq_frag_acc<NP>(ds + 8)};
      Frag<NP> pf[2];
      if constexpr (FIX) {
        pf[0] = gq_frag_acc<NP>(p);
        pf[1] = gq_frag_acc<NP>(p + 8);
      }
#pragma unroll
      for (int i = 0; i < OB; ++i) {
        if constexpr (NP == 1) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const gq_bf16x8 f = gq_frag_tr<1, D, PL>(Kt, ln, 32 * kb + 16 * u, i).p[0];
            acc[i] = gq_mfma(f, df[u].p[0], acc[i]);
            if constexpr (FIX) pk[i] = gq_mfma(f, pf[u].p[0], pk[i]);
          }
        } else {
          gq_f32x16 x = gq_zero();
          Frag<NP> kf[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            kf[u] = gq_frag_tr<NP, D, PL>(Kt, ln, 32 * kb + 16 * u, i);
            x = gq_mfma_small(kf[u], df[u], x);
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) x = gq_mfma(kf[u].p[0], df[u].p[0], x);
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][r] += x[r];
        }
      }
    }
  }

  if (qi >= a.Sq) return;
  // one part: the result, and D for the next kernel. Parts: this one's sums (of p k too), R and D'.
  constexpr bool PARTS = FIX || !REST;
  if (REST) rest = gq_sum_halves(rest);
  const size_t rows = (size_t)a.B * a.H * a.Sq;
  if (h == 0 && (!PARTS || a.splits == 1 || it.split == 0)) a.delta[at] = !PARTS || a.splits == 1 ? delta + rest : delta;
  if (FIX && h == 0 && a.splits > 1) a.part1[it.split * rows + at] = rest;
  T* drow = static_cast<T*>(a.dq) + ((long long)it.b * a.Sq + qi) * a.lddq + (long long)head * a.dk;
  const size_t prow = it.split * rows + ((size_t)it.b * a.Sq + qi) * a.H + head;
#pragma unroll
  for (int i = 0; i < OB; ++i)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      const int d = 32 * i + 8 * g4 + 4 * h;
      if (d >= a.dk) continue;
      float x[4], y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = acc[i][4 * g4 + j];
        if (FIX) {
          y[j] = live ? pk[i][4 * g4 + j] : 0.f;
          if (a.splits == 1) x[j] -= rest * y[j];
        }
        x[j] = live ? x[j] * a.scale : 0.f;
      }
      if (!PARTS || a.splits == 1) {
        gq_store4(drow, d, a.dk, x);
      } else {
        gq_store4(a.part0 + prow * (FIX ? 2 : 1) * a.dk, d, a.dk, x);
        if (FIX) gq_store4(a.part0 + (prow * 2 + 1) * a.dk, d, a.dk, y);
      }
    }
}

// The parts of dQ joined where R corrects it: 32 lanes a row. part0 [splits][B][Sq][H][scale sum dS' k | sum p k], part1
// [splits][B][H][Sq] R; delta D' in, D out.
template <typename T>
__global__ __launch_bounds__(256) void gqa_dq_join_kernel(GqaArgs a) {
  const long long rows = (long long)a.B * a.Sq * a.H, row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int d = 4 * (threadIdx.x & 31), head = (int)(row % a.H);
  const long long token = row / a.H, at = (token / a.Sq * a.H + head) * a.Sq + token % a.Sq;
  float rest = 0.f;
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) rest += a.part1[s * rows + at];
  if (d == 0) a.delta[at] += rest;
  if (d >= a.dk) return;
  float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float* p = a.part0 + (s * rows + row) * 2 * a.dk;
    float v[4], w[4];
    load_piece(p, d, a.dk, v);
    load_piece(p + a.dk, d, a.dk, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] += v[j];
      y[j] += w[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] -= a.scale * rest * y[j];
  gq_store4(static_cast<T*>(a.dq) + token * a.lddq + (long long)head * a.dk, d, a.dk, x);
}

// Distances that an LDS array holds beyond -M .. M on each side: a block that is not wholly M or more away reaches at
// most 62 further (and lane 63's place, which gets zeros, is one more).
constexpr int kSlack = 64;

// Where the scores of a query that has none start from: far enough below any others at every scale within 1e-30 .. 1e30.
constexpr float kUnseen = -3e38f;

// The sums of an accumulator's diagonals: lane i gets the sum of the values whose column less row is i - 31 (lane 63:
// zero). Rows 8 j + 0..3 are the registers 4 j .. 4 j + 3 of the lower half, 8 j + 4..7 of the upper. Each of four chains
// takes its eight rows, one after the other, into a row moved up by a lane a step, in 64 lanes of which the first 32 meet
// values; the four are then brought together 8 lanes apart.
__device__ __forceinline__ float diagonals(const float (&v)[16]) {
  float chain[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[4 * j + i]), 0u, false, false);
      lo[i] = x[0];  // the lower half's value and zeros
      hi[i] = x[1];  // the upper half's, moved down, and zeros
    }
    float c = __uint_as_float(lo[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i)  // wave_shr:1, zero into lane 0
      c = __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(c), 0x138, 0xf, 0xf, true)) +
          __uint_as_float(i < 4 ? lo[i] : hi[i - 4]);
    chain[j] = c;  // lane l + 7 - (row - 8 j); nothing from lane 39 on
  }
  const int lane = threadIdx.x & 63;
  float x = chain[3];
#pragma unroll
  for (int j = 0; j < 3; ++j)
    x += __uint_as_float(__builtin_amdgcn_ds_bpermute(4 * ((lane - 8 * (3 - j)) & 63), __float_as_uint(chain[j])));
  return x;
}

template <typename T, int D, int NQ, int NBUF>
struct DkvShape {
  static constexpr int NP = kPlanes<T>, KEYS = 128, BUF = 2 * NP * NQ * D;
  static constexpr size_t tile_bytes = (size_t)NBUF * BUF * 2;
  static size_t lds(bool dbias, int M) {
    return tile_bytes + (dbias ? (size_t)4 * (2 * M + 1 + 2 * kSlack) * 4 + 8 * 4 : 0);
  }
};

// BIAS: 0 none, 1 added, 2 added and its gradient wanted.
template <typename T, int D, int NQ, int NBUF, int BIAS, bool DMA>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kBwdWaves<T, D, DMA>))) void gqa_dkv_kernel(GqaArgs a) {
  using S = DkvShape<T, D, NQ, NBUF>;
  constexpr int NP = S::NP, KS = D / 16, OB = D / 32, QB = NQ / 32, PL = NQ * D;
  extern __shared__ __align__(16) uint16_t lds[];
  float* const far = reinterpret_cast<float*>(reinterpret_cast<char*>(lds) + S::tile_bytes);  // [4 waves][left, right]
  float* const dist = far + 8;                                                                  // [4 waves][W]
  const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5, wv = gq_wave();
  // Scores and dP start from -lse and -D in their accumulators; for the bias gradient, whose sums run over whole columns
  // of them, both are added afterwards as the dQ kernel does, so that the two kernels' dS agree: accumulators round
  // towards minus infinity, at the size of what they hold.
  constexpr bool INIT = BIAS != 2;
  const GqaItem it = gq_item(a, false);
  const GqaSample sm = gq_sample(a, it.b);
  const int key0 = it.tile * S::KEYS, k0 = key0 + wv * 32, key = k0 + l32;
  const int W = 2 * a.M + 1 + 2 * kSlack;
  const int g_beg = it.split / a.splits_q * a.heads_per_split, g_end = g_beg + a.heads_per_split;
  const int part_q = it.split % a.splits_q;
  // tiles of queries that see a key of this workgroup, and this part's share of them
  const int nqt = key0 < sm.kl ? (sm.ql + NQ - 1) / NQ : 0;
  const int first = a.causal ? min(nqt, max(0, key0 - sm.off) / NQ) : 0, count = nqt - first;
  const int q_beg = first + (int)((long long)count * part_q / a.splits_q);
  const int q_end = first + (int)((long long)count * (part_q + 1) / a.splits_q);

  Frag<NP> kf[KS], vf[KS];
  {
    const long long token = (long long)it.b * a.Sk + (key < sm.kl ? key : 0);
    const T* krow = static_cast<const T*>(a.k) + token * a.ldk + (long long)it.kvh * a.dk;
    const T* vrow = static_cast<const T*>(a.v) + token * a.ldv + (long long)it.kvh * a.dv;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      Eight<T> e, g;
      const int c = 16 * s + 8 * h;
      e.zero();
      g.zero();
      if (key < sm.kl && c < a.dk) e.load(krow, c, a.dk);
      if (key < sm.kl && c < a.dv) g.load(vrow, c, a.dv);
      kf[s] = gq_frag(e);
      vf[s] = gq_frag(g);
    }
  }
  GqaLane<D> ln;
  gq_f32x16 dk[OB], dv[OB];
#pragma unroll
  for (int i = 0; i < OB; ++i) dk[i] = dv[i] = gq_zero();

  std::conditional_t<DMA, GqaDma<D, NQ>, GqaTile<T, D, NQ>> qt, gt;
  if constexpr (DMA) {
    qt.init(a.ldq);
    gt.init(a.lddo);
  }
  // of the next tile's query l32 in each block of 32: what its scores and dP start from
  float s0_next[QB], dp0_next[QB];
  const T* qb0 = static_cast<const T*>(a.q) + (long long)it.b * a.Sq * a.ldq;
  const T* gb0 = static_cast<const T*>(a.dout) + (long long)it.b * a.Sq * a.lddo;
  auto fetch = [&](int g, int t, uint16_t* to) {
    const int head = it.kvh * a.G + g;
    if constexpr (DMA) {
      qt.issue(qb0 + (long long)head * a.dk, a.ldq, t * NQ, sm.ql, to);
      gt.issue(gb0 + (long long)head * a.dv, a.lddo, t * NQ, sm.ql, to + PL);
    } else {
      qt.fetch(qb0 + (long long)head * a.dk, a.ldq, t * NQ, sm.ql, a.dk);
      gt.fetch(gb0 + (long long)head * a.dv, a.lddo, t * NQ, sm.ql, a.dv);
    }
    const long long at = ((long long)it.b * a.H + head) * a.Sq;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const int q = t * NQ + 32 * qb + l32;
      s0_next[qb] = q < sm.ql ? a.lse[at + q] : -INFINITY;
      dp0_next[qb] = q < sm.ql ? -a.delta[at + q] : 0.f;
    }
  };
  if (q_beg < q_end) fetch(g_beg, q_beg, lds);
  const float inv_scale = 1.f / a.scale;
  int n = 0;  // tiles done
  for (int g = g_beg; g < g_end; ++g) {
    const int head = it.kvh * a.G + g;
    const float* bias = nullptr;
    float bias_l = 0.f, bias_r = 0.f, far_l = 0.f, far_r = 0.f;
    if (BIAS) {
      bias = a.bias + (size_t)head * (2 * a.M + 1) + a.M;
      bias_l = gq_bias(bias[-a.M]);
      bias_r = gq_bias(bias[a.M]);
    }
    float* mine = dist + wv * W + a.M + kSlack;
    if (BIAS == 2) {
      for (int i = threadIdx.x; i < 4 * W; i += 256) dist[i] = 0.f;
      __syncthreads();
    }
    for (int t = q_beg; t < q_end; ++t, ++n) {
      uint16_t* buf = lds + (NBUF == 2 ? (n & 1) * S::BUF : 0);
      if (NBUF == 1 && n) __syncthreads();
      if constexpr (!DMA) {
        qt.stash(buf);
        gt.stash(buf + NP * PL);
      }
      float s0[QB], dp0[QB];
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        // -lse in the scores' own units; a query past the sample's, or one that saw no key: every p is 0
        s0[qb] = s0_next[qb] == -INFINITY ? kUnseen : -s0_next[qb] * inv_scale;
        dp0[qb] = dp0_next[qb];
      }
      uint16_t* next = lds + (NBUF == 2 ? ((n + 1) & 1) * S::BUF : 0);
      if constexpr (DMA) {
        gq_dma_wait();
        __syncthreads();
      }
      if (t + 1 < q_end) fetch(g, t + 1, next);
      else if (g + 1 < g_end) fetch(g + 1, q_beg, next);
      if constexpr (!DMA) __syncthreads();
      const uint16_t *Qt = buf, *Gt = buf + NP * PL;
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        const int q0 = t * NQ + 32 * qb;
        if (q0 >= sm.ql || k0 >= sm.kl || (a.causal && k0 > q0 + 31 + sm.off)) continue;
        ln.renew();
        gq_f32x16 s = INIT ? gq_rows(s0[qb], h) : gq_zero(), dp = INIT ? gq_rows(dp0[qb], h) : gq_zero();
        {
          gq_f32x16 lo = gq_zero(), lo2 = gq_zero();
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const Frag<NP> f = gq_frag_row<NP, D, PL>(Qt, ln, qb * 32, ks);
            if constexpr (NP == 3) lo = gq_mfma_small(f, kf[ks], lo);
            s = gq_mfma(f.p[0], kf[ks].p[0], s);
          }
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const Frag<NP> f = gq_frag_row<NP, D, PL>(Gt, ln, qb * 32, ks);
            if constexpr (NP == 3) lo2 = gq_mfma_small(f, vf[ks], lo2);
            dp = gq_mfma(f.p[0], vf[ks].p[0], dp);
          }
          if constexpr (NP == 3) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              s[r] += lo[r];
              dp[r] += lo2[r];
            }
          }
        }
        float mul = a.c, add = 0.f;
        int side = 0;  // of the block's distances: all <= -M, all >= M, or near
        if (BIAS) {
          if (k0 + 31 - (q0 + sm.off) <= -a.M) {
            add = bias_l;
            side = -1;
          } else if (k0 - (q0 + 31 + sm.off) >= a.M) {
            add = bias_r;
            side = 1;
          } else {
            mul = 1.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int d = key - (q0 + gq_row(r, h) + sm.off);
              s[r] = fmaf(s[r], a.c, gq_bias(bias[min(max(d, -a.M), a.M)]));
            }
          }
        }
        if (k0 + 31 >= sm.kl || (a.causal && k0 + 31 > q0 + sm.off)) {
          // queries past the sample's are no matter here: their scores start from kUnseen
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (key >= sm.kl || (a.causal && key > q0 + gq_row(r, h) + sm.off)) {
              s[r] = -INFINITY;
              dp[r] = 0.f;
            }
        }
        float p[16], ds[16];
        if constexpr (INIT) {
#pragma unroll
          for (int r = 0; r < 16; ++r) p[r] = __builtin_amdgcn_exp2f(fmaf(s[r], mul, add));
#pragma unroll
          for (int r = 0; r < 16; ++r) ds[r] = p[r] * dp[r];
        } else {
          const gq_f32x16 ls = gq_rows(s0[qb] == kUnseen ? -1e30f : s0[qb] * a.c, h);  // finite pieces
#pragma unroll
          for (int r = 0; r < 16; ++r) p[r] = __builtin_amdgcn_exp2f(fmaf(s[r], mul, add + ls[r]));
          const gq_f32x16 de = gq_rows(dp0[qb], h);
#pragma unroll
          for (int r = 0; r < 16; ++r) ds[r] = p[r] * (dp[r] + de[r]);
        }
        if (BIAS == 2) {
          if (side == 0) {
            const float x = diagonals(ds);
            // lane 63's is zero, and its place within the slack
            mine[k0 - q0 - sm.off - 31 + lane] += x;
          } else {
            float x = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) x += ds[r];
            if (side < 0) far_l += x;
            else far_r += x;
          }
        }
        const Frag<NP> pf[2] = {gq_frag_acc<NP>(p), gq_frag_acc<NP>(p + 8)};
        const Frag<NP> df[2] = {gq_frag_acc<NP>(ds), gq_frag_acc<NP>(ds + 8)};
#pragma unroll
        for (int i = 0; i < OB; ++i) {
          if constexpr (NP == 1) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              dv[i] = gq_mfma(gq_frag_tr<1, D, PL>(Gt, ln, 32 * qb + 16 * u, i).p[0], pf[u].p[0], dv[i]);
              dk[i] = gq_mfma(gq_frag_tr<1, D, PL>(Qt, ln, 32 * qb + 16 * u, i).p[0], df[u].p[0], dk[i]);
            }
          } else {
#pragma unroll
            for (int which = 0; which < 2; ++which) {
              gq_f32x16 x = gq_zero();
              Frag<NP> f[2];
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                f[u] = gq_frag_tr<NP, D, PL>(which ? Qt : Gt, ln, 32 * qb + 16 * u, i);
                x = gq_mfma_small(f[u], which ? df[u] : pf[u], x);
              }
#pragma unroll
              for (int u = 0; u < 2; ++u) x = gq_mfma(f[u].p[0], which ? df[u].p[0] : pf[u].p[0], x);
#pragma unroll
              for (int r = 0; r < 16; ++r) (which ? dk : dv)[i][r] += x[r];
            }
          }
        }
      }
    }
    if (BIAS == 2) {
      far_l = wave_sum(far_l);
      far_r = wave_sum(far_r);
      if (lane == 0) {
        far[2 * wv] = far_l;
        far[2 * wv + 1] = far_r;
      }
      __syncthreads();
      const int n_out = 2 * a.M + 1;
      float* part = a.dbias_part +
                    ((((long long)it.b * a.H + head) * a.tiles + it.tile) * a.splits_q + part_q) * n_out;
      auto fold = [&](int e) { return (dist[e] + dist[W + e]) + (dist[2 * W + e] + dist[3 * W + e]); };
      for (int i = 1 + threadIdx.x; i < n_out - 1; i += 256) part[i] = fold(i + kSlack);
      // the ends take every distance beyond them: a wave each
      if (wv < 2) {
        const int at = wv == 0 ? 0 : W - kSlack - 1;
        const float x = wave_sum(fold(at + lane) + (lane == 0 ? fold(at + kSlack) : 0.f));
        if (lane == 0) part[wv == 0 ? 0 : n_out - 1] = x + ((far[wv] + far[2 + wv]) + (far[4 + wv] + far[6 + wv]));
      }
      __syncthreads();  // before the next head's arrays are cleared
    }
  }

  if (key >= a.Sk) return;
  const long long token = (long long)it.b * a.Sk + key;
  const long long prow = (((long long)it.split * a.B * a.Sk + token) * a.KV + it.kvh);
#pragma unroll
  for (int i = 0; i < OB; ++i)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      const int d = 32 * i + 8 * g4 + 4 * h;
      float x[4], y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = dk[i][4 * g4 + j] * a.scale;
        y[j] = dv[i][4 * g4 + j];
      }
      if (a.splits == 1) {
        if (d < a.dk) gq_store4(static_cast<T*>(a.dkey) + token * a.lddk + (long long)it.kvh * a.dk, d, a.dk, x);
        if (d < a.dv) gq_store4(static_cast<T*>(a.dval) + token * a.lddv + (long long)it.kvh * a.dv, d, a.dv, y);
      } else {
        if (d < a.dk) gq_store4(a.part0 + prow * a.dk, d, a.dk, x);
        if (d < a.dv) gq_store4(a.part1 + prow * a.dv, d, a.dv, y);
      }
    }
}

// dbias[h][i] = beta dbias[h][i] + the parts of head h, in f64 and a fixed order: part [B][H][per][n].
__global__ __launch_bounds__(1024) void gqa_dbias_kernel(int B, int H, int per, int n, const float* __restrict__ part,
                                                         float beta, float* dbias) {
  __shared__ double red[16][64];
  const int l = threadIdx.x & 63, wv = threadIdx.x >> 6, i = blockIdx.x * 64 + l, hd = blockIdx.y;
  double s = 0.0;
  if (i < n)
    for (long long r = wv; r < (long long)B * per; r += 16)
      s += (double)part[((r / per * H + hd) * per + r % per) * n + i];
  red[wv][l] = s;
  __syncthreads();
  if (wv != 0 || i >= n) return;
  s = 0.0;
#pragma unroll
  for (int w = 0; w < 16; ++w) s += red[w][l];
  float* o = dbias + (size_t)hd * n + i;
  *o = (float)(s + (beta != 0.f ? (double)*o : 0.0));
}

// The kernels of one head width.
struct BwdShape {
  const void *dq[2], *dq_few[2];  // dq_few: null for fp32
  const void* dkv[3];
  size_t dq_lds;
  size_t (*dkv_lds)(bool, int);
};
template <typename T, int D, int NK, int NBK, int NQ, int NBQ, bool DMA = false>
BwdShape bwd_shape() {
  const void *few = nullptr, *few_bias = nullptr;
  if constexpr (sizeof(T) == 2) {
    few = (const void*)gqa_dq_kernel<T, D, NK, NBK, false, DMA, true>;
    few_bias = (const void*)gqa_dq_kernel<T, D, NK, NBK, true, DMA, true>;
  }
  return {{(const void*)gqa_dq_kernel<T, D, NK, NBK, false, DMA, false>,
           (const void*)gqa_dq_kernel<T, D, NK, NBK, true, DMA, false>},
          {few, few_bias},
          {(const void*)gqa_dkv_kernel<T, D, NQ, NBQ, 0, DMA>, (const void*)gqa_dkv_kernel<T, D, NQ, NBQ, 1, DMA>,
           (const void*)gqa_dkv_kernel<T, D, NQ, NBQ, 2, DMA>},
          DqShape<T, D, NK, NBK>::lds, DkvShape<T, D, NQ, NBQ>::lds};
}
// Tiles of keys (dQ) and of queries (dK, dV), two buffers each: 64 rows where a workgroup's LDS and registers hold them
// beside a second workgroup's. Measured (forward and backward): 4 x 4096 tokens, d 128 bf16: query tiles of 64 1583 us, of
// 32 1649; key tiles of 64 no better than 32 (1647). 2 x 2048, d 64 bf16: 276, with 32-row tiles 295. fp32, d 128, 21
// samples of 1520 queries and 405 keys: two buffers of 32 rows 1595, one 1660. Direct tiles (gq_dma_fits): 4 x 4096, d 128
// 1627 us, through registers 2260; 2 x 2048, d 64 276 and 278.
template <typename T>
BwdShape pick_bwd(int d, bool dma) {
  if constexpr (sizeof(T) == 2) {
    if (dma && d == 32) return bwd_shape<T, 32, 64, 2, 64, 2, true>();
    if (dma && d == 64) return bwd_shape<T, 64, 64, 2, 64, 2, true>();
    if (dma && d == 128) return bwd_shape<T, 128, 32, 2, 64, 2, true>();
    if (d <= 32) return bwd_shape<T, 32, 64, 2, 32, 2>();
    if (d <= 64) return bwd_shape<T, 64, 64, 2, 32, 2>();
    return bwd_shape<T, 128, 32, 2, 32, 2>();
  } else {
    if (d <= 32) return bwd_shape<T, 32, 32, 2, 32, 2>();
    if (d <= 64) return bwd_shape<T, 64, 32, 2, 32, 2>();
    return bwd_shape<T, 128, 32, 2, 32, 2>();
  }
}

int launch(const void* fn, size_t blocks, size_t lds, GqaArgs* a, hipStream_t s, const char* name) {
  TALOS_REQUIRE(blocks <= 0x7fffffffu, TALOS_ERR_UNSUPPORTED, "%s: %zu workgroups", name, blocks);
  if (lds > 65536) TALOS_HIP(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  void* args[] = {a};
  return hip_status(hipLaunchKernel(fn, dim3((unsigned)blocks), dim3(256), args, lds, s), name);
}

// Keys up to which a workgroup of bf16 rows has its dQ corrected by R. The error of dQ, 4 x 4096 causal tokens: 2.36e-3 with
// any of 64 to 512 (2.45e-3 uncorrected), 672 ragged ones 2.35e-3 (2.52e-3), 3799 queries of 781 keys 2.39e-3 with 64 or 128,
// 2.37e-3 with 256; time of the first 1447, 1459, 1467, 1476 us for 64, 128, 256, 512.
constexpr int kFewKeys = 128;
constexpr int kDbiasMaxDistance = 512;  // four arrays of 2 M + 129 floats beside the tiles in a workgroup's LDS
// Workgroups that fill the device: two a compute unit (4 x 4096 tokens, d 128: 1627 us; for 256 1968, for 1024 1650; 2 x
// 2048, d 64: 276, 277, 362).
constexpr long long kFill = 512;

template <typename T>
int bwd(const char* fn, const talos_gqa_cfg* cfg, const int32_t* q_lens, const int32_t* k_lens, const float* bias,
        const T* q, long long ld_q, const T* k, long long ld_k, const T* v, long long ld_v, const T* o, long long ld_o,
        const float* lse, const T* dout, long long ld_do, T* dq, long long ld_dq, T* dk, long long ld_dk, T* dv,
        long long ld_dv, float beta_bias, float* dbias, hipStream_t s) {
  int rc = gqa_check(fn, cfg, bias, q, ld_q, k, ld_k, v, ld_v, o, ld_o, lse);
  if (rc) return rc;
  GqaArgs a = gqa_args(cfg, q_lens, k_lens, bias, q, ld_q, k, ld_k, v, ld_v);
  const bool queries = a.B > 0 && a.Sq > 0, keys = a.B > 0 && a.Sk > 0;
  TALOS_REQUIRE((!queries || (dout && dq)) && (!keys || (dk && dv)), TALOS_ERR_NULL, "%s: null dout, dq, dk or dv", fn);
  TALOS_REQUIRE(ld_do >= (long long)a.H * a.dv && ld_dq >= (long long)a.H * a.dk && ld_dk >= (long long)a.KV * a.dk &&
                    ld_dv >= (long long)a.KV * a.dv,
                TALOS_ERR_SHAPE, "%s: a gradient row stride is smaller than heads * dim", fn);
  TALOS_REQUIRE(!dbias || bias, TALOS_ERR_NULL, "%s: dbias without bias", fn);
  TALOS_REQUIRE(beta_bias == 0.f || beta_bias == 1.f, TALOS_ERR_UNSUPPORTED, "%s: beta_bias must be 0 or 1", fn);
  TALOS_REQUIRE(!dbias || a.M <= kDbiasMaxDistance, TALOS_ERR_UNSUPPORTED,
                "%s: the bias gradient takes max_distance <= %d, not %d", fn, kDbiasMaxDistance, a.M);
  TALOS_REQUIRE(!dbias || a.H <= 65535, TALOS_ERR_UNSUPPORTED, "%s: the bias gradient takes at most 65535 heads", fn);
  TALOS_DEVICE();
  a.o = o;
  a.ldo = ld_o;
  a.lse = const_cast<float*>(lse);
  a.dout = dout;
  a.lddo = ld_do;
  a.dq = dq;
  a.lddq = ld_dq;
  a.dkey = dk;
  a.lddk = ld_dk;
  a.dval = dv;
  a.lddv = ld_dv;
  const bool dma = a.dk == a.dv && gq_dma_fits(q, ld_q) && gq_dma_fits(k, ld_k) && gq_dma_fits(v, ld_v) &&
                   gq_dma_fits(dout, ld_do);
  const BwdShape shape = pick_bwd<T>(std::max(a.dk, a.dv), dma);

  // Parts of the key loop (dQ), of the heads and then of the query loop (dK, dV) where there is too little to do: of at
  // least 256 keys or queries (22 samples of 247 queries and 79 keys, fp32 d 56: 168 us, with parts of 128 188).
  const long long pairs = (long long)a.B * a.KV;
  const long long q_tiles = ((long long)a.G * a.Sq + 127) / 128, k_tiles = (a.Sk + 127) / 128;
  const long long q_base = pairs * q_tiles, k_base = pairs * k_tiles;
  const long long fill = kFill / (std::max(a.dk, a.dv) > 64 && !dma ? 2 : 1);  // where a wave has a SIMD to itself
  long long sp_k = q_base ? std::min((fill + q_base - 1) / q_base, ((long long)a.Sk + 255) / 256) : 1;
  sp_k = std::max(1ll, sp_k);
  long long sp_h = 1, sp_q = 1;
  // a causal key tile's share of the work, and a sample's, differ: twice the parts even them out (4 x 4096, d 128: 1627 us,
  // 1953 without)
  const long long fill_k = a.causal || q_lens || k_lens ? 2 * fill : fill;
  if (k_base && k_base < fill_k) {
    const long long want = (fill_k + k_base - 1) / k_base;
    for (long long d = 1; d <= a.G; ++d)  // the least divisor of the group that is enough, or the whole group
      if (a.G % d == 0 && (d >= want || d == a.G)) {
        sp_h = d;
        break;
      }
    sp_q = std::max(1ll, std::min((want + sp_h - 1) / sp_h, ((long long)a.Sq + 255) / 256));
  }
  constexpr bool fix = sizeof(T) == 2;
  const size_t dq_part = sp_k > 1 ? (size_t)sp_k * a.B * a.Sq * a.H * (fix ? 2 * a.dk + 1 : a.dk) : 0;
  const size_t kv_part = sp_h * sp_q > 1 ? (size_t)(sp_h * sp_q) * a.B * a.Sk * a.KV * (a.dk + a.dv) : 0;
  const size_t n_delta = ((size_t)a.B * a.H * a.Sq + 63) & ~(size_t)63;
  const size_t n_bias = dbias && queries ? (size_t)a.B * a.H * k_tiles * sp_q * (2 * a.M + 1) : 0;
  EntryScratch ws;
  rc = ws.acquire((n_delta + std::max(dq_part, kv_part) + n_bias) * sizeof(float), s);
  if (rc) return rc;
  a.delta = static_cast<float*>(ws.ptr);
  float* parts = a.delta + n_delta;
  a.dbias_part = parts + std::max(dq_part, kv_part);
  if (queries) {
    a.tiles = (int)q_tiles;
    a.splits = (int)sp_k;
    a.part0 = parts;
    a.part1 = parts + (size_t)sp_k * a.B * a.Sq * a.H * 2 * a.dk;  // where R is kept
    // fp32, or bf16 workgroups by the keys that their rows see (those with parts are few and see little each)
    a.few = sp_k > 1 ? INT_MAX : kFewKeys;
    const bool some = !fix || a.Sk > a.few, few = fix && (!some || a.causal || q_lens || k_lens);
    if (some) rc = launch(shape.dq[bias ? 1 : 0], q_base * sp_k, shape.dq_lds, &a, s, "gqa_dq_kernel");
    if (!rc && few) rc = launch(shape.dq_few[bias ? 1 : 0], q_base * sp_k, shape.dq_lds, &a, s, "gqa_dq_kernel");
    if (!rc && sp_k > 1) {
      if constexpr (fix) {
        hipLaunchKernelGGL(gqa_dq_join_kernel<T>, dim3(ceil_div((size_t)a.B * a.Sq * a.H, 8)), dim3(256), 0, s, a);
        rc = launch_status("gqa_dq_join_kernel");
      } else {
        rc = gqa_join_launch<T>((int)sp_k, (size_t)a.B * a.Sq, a.H * a.dk, parts, dq, ld_dq, s);
      }
    }
  }
  if (!rc && keys) {
    a.tiles = (int)k_tiles;
    a.splits = (int)(sp_h * sp_q);
    a.splits_q = (int)sp_q;
    a.heads_per_split = (int)(a.G / sp_h);
    a.part0 = parts;
    a.part1 = parts + (size_t)a.splits * a.B * a.Sk * a.KV * a.dk;
    const bool sums = dbias && queries;
    rc = launch(shape.dkv[sums ? 2 : bias ? 1 : 0], k_base * a.splits, shape.dkv_lds(sums, a.M), &a, s, "gqa_dkv_kernel");
    if (!rc && a.splits > 1) {
      rc = gqa_join_launch<T>(a.splits, (size_t)a.B * a.Sk, a.KV * a.dk, a.part0, dk, ld_dk, s);
      if (!rc) rc = gqa_join_launch<T>(a.splits, (size_t)a.B * a.Sk, a.KV * a.dv, a.part1, dv, ld_dv, s);
    }
  }
  if (!rc && dbias) {
    const int n = 2 * a.M + 1, per = queries && keys ? (int)(k_tiles * sp_q) : 0;
    hipLaunchKernelGGL(gqa_dbias_kernel, dim3(ceil_div(n, 64), a.H), dim3(1024), 0, s, per ? a.B : 0, a.H, std::max(per, 1), n,
                       a.dbias_part, beta_bias, dbias);
    rc = launch_status("gqa_dbias_kernel");
  }
  const int rel = ws.release();
  return entry_done(rc ? rc : rel, s);
}

}  // namespace
}  // namespace talos

using namespace talos;

extern "C" {

int talos_gqa_bwd_f32(const talos_gqa_cfg* cfg, const int32_t* q_lens, const int32_t* k_lens, const float* bias,
                      const float* q, long long ld_q, const float* k, long long ld_k, const float* v, long long ld_v,
                      const float* o, long long ld_o, const float* lse, const float* dout, long long ld_do, float* dq,
                      long long ld_dq, float* dk, long long ld_dk, float* dv, long long ld_dv, float beta_bias,
                      float* dbias, talos_stream_t stream) {
  return bwd<float>(__func__, cfg, q_lens, k_lens, bias, q, ld_q, k, ld_k, v, ld_v, o, ld_o, lse, dout, ld_do, dq, ld_dq,
                    dk, ld_dk, dv, ld_dv, beta_bias, dbias, as_stream(stream));
}
int talos_gqa_bwd_bf16(const talos_gqa_cfg* cfg, const int32_t* q_lens, const int32_t* k_lens, const float* bias,
                       const talos_bf16* q, long long ld_q, const talos_bf16* k, long long ld_k, const talos_bf16* v,
                       long long ld_v, const talos_bf16* o, long long ld_o, const float* lse, const talos_bf16* dout,
                       long long ld_do, talos_bf16* dq, long long ld_dq, talos_bf16* dk, long long ld_dk,
                       talos_bf16* dv, long long ld_dv, float beta_bias, float* dbias, talos_stream_t stream) {
  return bwd<Bf16>(__func__, cfg, q_lens, k_lens, bias, reinterpret_cast<const Bf16*>(q), ld_q,
                   reinterpret_cast<const Bf16*>(k), ld_k, reinterpret_cast<const Bf16*>(v), ld_v,
                   reinterpret_cast<const Bf16*>(o), ld_o, lse, reinterpret_cast<const Bf16*>(dout), ld_do,
                   reinterpret_cast<Bf16*>(dq), ld_dq, reinterpret_cast<Bf16*>(dk), ld_dk, reinterpret_cast<Bf16*>(dv),
                   ld_dv, beta_bias, dbias, as_stream(stream));
}

}  // extern "C"
