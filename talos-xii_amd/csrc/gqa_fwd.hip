// gqa_fwd.hip -- grouped-query attention, forward: one pass over the keys with a running maximum and sum.
//
// The queries of a group's G heads that share a key head are rows of one matrix (row r is query r / G of head
// r % G), so a key tile in LDS serves all of them. A wave holds 32 rows: their q as B operands, S^T = K Q^T of a
// block of keys (rows of a lane are keys, its column one query), the softmax along registers, and O^T += V^T P^T
// with P^T straight from the accumulator. Scores are in units of log 2, c = scale log2(e):
//   p = exp2(c s + b - m),  l += p,  O^T += v p,   o = O / l,  lse = (m + log2 l) ln 2
// m is the running maximum, raised (and O, l scaled) only when a row exceeds it by 2^8: p then stays below 256 in
// fp32, where any factor is exact enough, and most tiles scale nothing.
//
// Key blocks that every row of a wave sees whole take no comparison; only the blocks at a causal edge or a
// sample's end are masked. A bias by distance is one constant a row where the whole block is at least M away.
//
// Few rows (G q_len <= 32: decoding) leave three of four waves without rows: there the four waves take different
// keys of a tile four times as long, and their results are joined in LDS. Few workgroups: the keys are cut into
// parts, each with its own maximum and sum, joined by a second kernel.
#include <algorithm>
#include <type_traits>

#include "gqa.hpp"

namespace talos {

namespace {

template <typename T, int D, int NK, int KW, int NBUF>
struct FwdShape {
  static constexpr int NP = kPlanes<T>, TK = NK * KW, RW = 4 / KW, ROWS = 32 * RW;
  static constexpr int BUF = 2 * NP * TK * D;  // bf16 values of one buffer: K planes, V planes
  static constexpr size_t join_bytes = KW == 1 ? 0 : (size_t)RW * KW * (D * 32 + 2 * 64) * 4;
  static constexpr size_t lds = std::max((size_t)NBUF * BUF * 2, join_bytes);
};

// Two waves a SIMD (a wave's softmax beside another's products): 256 registers a lane, which the bf16 kernels and
// the fp32 ones to 64 columns fit; with no such bound the compiler keeps accumulators in the other register file and
// moves them for every tile (forward and backward, 4 x 4096 tokens, d 128 bf16: 1627 us, unbound 2538; 8 ragged samples of
// up to 1000, d 64 fp32: 320, 357).
template <typename T, int D>
constexpr int kFwdWaves = sizeof(T) == 4 && D == 128 ? 1 : 2;

// BIAS: by distance. DMA: bf16 tiles go from memory to LDS directly.
template <typename T, int D, int NK, int KW, int NBUF, bool BIAS, bool DMA>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kFwdWaves<T, D>))) void gqa_fwd_kernel(GqaArgs a) {
  static_assert(!DMA || (sizeof(T) == 2 && (NBUF == 2 || KW > 1)), "direct tiles are bf16, shared ones land in the other buffer");
  using S = FwdShape<T, D, NK, KW, NBUF>;
  constexpr int NP = S::NP, TK = S::TK, KS = D / 16, OB = D / 32, KB = NK / 32, PL = TK * D;
  extern __shared__ __align__(16) uint16_t lds[];
  const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5, wv = gq_wave();
  const int wr = wv / KW, kw = wv % KW;
  const GqaItem it = gq_item(a, true);
  const GqaSample sm = gq_sample(a, it.b);
  const int G = a.G;
  // this wave's rows
  const int row0 = it.tile * S::ROWS + wr * 32, row = row0 + l32;
  const int qi = row / G, head = it.kvh * G + row % G;
  const bool live = qi < sm.ql;
  const int lim = !live ? 0 : a.causal ? min(sm.kl, qi + sm.off + 1) : sm.kl;  // keys that the row sees
  // of the wave's live rows: the first sees least, the last most
  const int q_lo = row0 / G, q_hi = min((row0 + 31) / G, sm.ql - 1);
  const int lim_lo = a.causal ? min(sm.kl, q_lo + sm.off + 1) : sm.kl;
  const int lim_hi = q_lo >= sm.ql ? 0 : a.causal ? min(sm.kl, q_hi + sm.off + 1) : sm.kl;
  // of the workgroup's
  const int wg_lo = it.tile * S::ROWS / G, wg_hi = min((it.tile * S::ROWS + S::ROWS - 1) / G, sm.ql - 1);
  const int kend = wg_lo >= sm.ql ? 0 : a.causal ? max(0, min(sm.kl, wg_hi + sm.off + 1)) : sm.kl;
  const int ntile = (kend + TK - 1) / TK;
  const int t_beg = (int)((long long)ntile * it.split / a.splits), t_end = (int)((long long)ntile * (it.split + 1) / a.splits);

  const T* kbase = static_cast<const T*>(a.k) + (long long)it.b * a.Sk * a.ldk + (long long)it.kvh * a.dk;
  const T* vbase = static_cast<const T*>(a.v) + (long long)it.b * a.Sk * a.ldv + (long long)it.kvh * a.dv;
  // few rows and direct tiles: each wave streams the tiles of its own keys and meets the others only at the end
  constexpr bool ALONE = DMA && KW > 1;
  std::conditional_t<DMA, GqaDma<D, ALONE ? NK : TK, ALONE ? 1 : 4>, GqaTile<T, D, TK>> kt, vt;
  if constexpr (DMA) {
    kt.init(a.ldk);
    vt.init(a.ldv);
  }
  if constexpr (ALONE) {
    if (t_beg < t_end && t_beg * TK + kw * NK < lim_hi) {
      kt.issue(kbase, a.ldk, t_beg * TK + kw * NK, sm.kl, lds + kw * NK * D);
      vt.issue(vbase, a.ldv, t_beg * TK + kw * NK, sm.kl, lds + PL + kw * NK * D);
    }
  } else if (t_beg < t_end) {
    if constexpr (DMA) {
      uint16_t* buf = lds + (t_beg & 1) * S::BUF;
      kt.issue(kbase, a.ldk, t_beg * TK, sm.kl, buf);
      vt.issue(vbase, a.ldv, t_beg * TK, sm.kl, buf + PL);
    } else {
      kt.fetch(kbase, a.ldk, t_beg * TK, sm.kl, a.dk);
      vt.fetch(vbase, a.ldv, t_beg * TK, sm.kl, a.dv);
    }
  }
  Frag<NP> qf[KS];
  {
    const T* qrow = static_cast<const T*>(a.q) + ((long long)it.b * a.Sq + (live ? qi : 0)) * a.ldq + (long long)head * a.dk;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      Eight<T> e;
      const int c = 16 * s + 8 * h;
      if (live && c < a.dk) e.load(qrow, c, a.dk);
      else e.zero();
      qf[s] = gq_frag(e);
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
  float m = -INFINITY, l = 0.f;
  gq_f32x16 acc[OB];
#pragma unroll
  for (int i = 0; i < OB; ++i) acc[i] = gq_zero();

  for (int t = t_beg; t < t_end; ++t) {
    uint16_t* buf = lds + (NBUF == 2 ? (t & 1) * S::BUF : 0);
    const int k0 = t * TK + kw * NK;  // this wave's keys
    const bool more = t + 1 < t_end && k0 + TK < lim_hi;
    if constexpr (ALONE) {
      // in flight, in order: K of this tile, V of this tile
      if (k0 < lim_hi) gq_dma_wait<decltype(vt)::PER>();
    } else if constexpr (DMA) {
      gq_dma_wait();
      __syncthreads();  // tile t is here, and the other buffer's readers are done
      if (t + 1 < t_end) {
        uint16_t* next = lds + ((t + 1) & 1) * S::BUF;
        kt.issue(kbase, a.ldk, (t + 1) * TK, sm.kl, next);
        vt.issue(vbase, a.ldv, (t + 1) * TK, sm.kl, next + PL);
      }
    } else {
      if (NBUF == 1 && t != t_beg) __syncthreads();  // the last tile's readers are done
      kt.stash(buf);
      vt.stash(buf + NP * PL);
      if (t + 1 < t_end) {
        kt.fetch(kbase, a.ldk, (t + 1) * TK, sm.kl, a.dk);
        vt.fetch(vbase, a.ldv, (t + 1) * TK, sm.kl, a.dv);
      }
      __syncthreads();
    }
    if (k0 >= lim_hi) continue;
    const uint16_t *Kt = buf + kw * NK * D, *Vt = buf + NP * PL + kw * NK * D;
    ln.renew();
    gq_f32x16 s[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      gq_f32x16 hi = gq_zero(), lo = gq_zero();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const Frag<NP> kf = gq_frag_row<NP, D, PL>(Kt, ln, kb * 32, ks);
        if constexpr (NP == 3) lo = gq_mfma_small(kf, qf[ks], lo);
        hi = gq_mfma(kf.p[0], qf[ks].p[0], hi);
      }
      if constexpr (NP == 3) {
#pragma unroll
        for (int r = 0; r < 16; ++r) hi[r] += lo[r];
      }
      s[kb] = hi;
    }
    if constexpr (ALONE) {
      gq_reads_done();
      if (more) kt.issue(kbase, a.ldk, k0 + TK, sm.kl, lds + kw * NK * D);
    }
    // the first fragments of V: on their way from LDS beside the softmax
    constexpr int PRE = NP == 1 && !ALONE ? (2 < OB ? 2 : OB) : 0;
    Frag<NP> early[PRE ? PRE : 1][2 * KB];
#pragma unroll
    for (int i = 0; i < PRE; ++i)
#pragma unroll
      for (int u = 0; u < 2 * KB; ++u) early[i][u] = gq_frag_tr<NP, D, PL>(Vt, ln, 16 * u, i);
    // scores in units of log 2, bias and mask included, less nothing yet; their maximum
    float add = 0.f;  // what every score of the row still lacks
    bool raw = true;  // s still lacks the factor c too
    if (BIAS) {
      if (k0 + NK - 1 - (q_lo + sm.off) <= -a.M) {
        add = bias_l;
      } else if (k0 - (q_hi + sm.off) >= a.M) {
        add = bias_r;
      } else {
        raw = false;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int d = k0 + kb * 32 + gq_row(r, h) - pos;
            s[kb][r] = fmaf(s[kb][r], a.c, gq_bias(bias[min(max(d, -a.M), a.M)]));
          }
      }
    }
    if (k0 + NK > lim_lo) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (k0 + kb * 32 + gq_row(r, h) >= lim) s[kb][r] = -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[kb][r]);
    top = gq_max_halves(top);
    const float mul = raw ? a.c : 1.f;
    top = fmaf(top, mul, add);
    if (__any(top > m + 8.f)) {
      const float mn = fmaxf(m, top);
      const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= alpha;
#pragma unroll
      for (int i = 0; i < OB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] *= alpha;
      m = mn;
    }
    const float sub = add - (m == -INFINITY ? 0.f : m);
    float sum = 0.f;
    Frag<NP> pf[2 * KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = __builtin_amdgcn_exp2f(fmaf(s[kb][r], mul, sub));
        sum += p[r];
      }
      pf[2 * kb] = gq_frag_acc<NP>(p);
      pf[2 * kb + 1] = gq_frag_acc<NP>(p + 8);
    }
    l += sum;
    if constexpr (ALONE) {
      if (more) gq_dma_wait<decltype(kt)::PER>();
      else gq_dma_wait();
    }
#pragma unroll
    for (int i = 0; i < OB; ++i) {
      if constexpr (NP == 1) {
#pragma unroll
        for (int u = 0; u < 2 * KB; ++u)
          acc[i] = gq_mfma(i < PRE ? early[i < PRE ? i : 0][u].p[0] : gq_frag_tr<1, D, PL>(Vt, ln, 16 * u, i).p[0], pf[u].p[0], acc[i]);
      } else {
        // the tile's product by itself, the small pairs first, then one fp32 addition
        gq_f32x16 x = gq_zero();
        Frag<NP> vf[2 * KB];
#pragma unroll
        for (int u = 0; u < 2 * KB; ++u) {
          vf[u] = gq_frag_tr<NP, D, PL>(Vt, ln, 16 * u, i);
          x = gq_mfma_small(vf[u], pf[u], x);
        }
#pragma unroll
        for (int u = 0; u < 2 * KB; ++u) x = gq_mfma(vf[u].p[0], pf[u].p[0], x);
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] += x[r];
      }
    }
    if constexpr (ALONE) {
      gq_reads_done();
      if (more) vt.issue(vbase, a.ldv, k0 + TK, sm.kl, lds + PL + kw * NK * D);
    }
  }
  l = gq_sum_halves(l);

  if constexpr (KW > 1) {
    // the waves of a row group join: each takes every KW-th block of 32 columns
    float* f = reinterpret_cast<float*>(lds);
    float* stat = f + S::RW * KW * D * 32;
    __syncthreads();
    const int w = wr * KW;
#pragma unroll
    for (int i = 0; i < OB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) f[(((w + kw) * OB + i) * 16 + r) * 64 + lane] = acc[i][r];
    stat[(w + kw) * 128 + lane] = m;
    stat[(w + kw) * 128 + 64 + lane] = l;
    __syncthreads();
    float mj = -INFINITY;
#pragma unroll
    for (int j = 0; j < KW; ++j) mj = fmaxf(mj, stat[(w + j) * 128 + lane]);
    float sc[KW];
    l = 0.f;
#pragma unroll
    for (int j = 0; j < KW; ++j) {
      const float x = stat[(w + j) * 128 + lane];
      sc[j] = x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x - mj);
      l += sc[j] * stat[(w + j) * 128 + 64 + lane];
    }
    m = mj;
#pragma unroll
    for (int i = 0; i < OB; ++i)
      if (i % KW == kw)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float x = 0.f;
#pragma unroll
          for (int j = 0; j < KW; ++j) x += sc[j] * f[(((w + j) * OB + i) * 16 + r) * 64 + lane];
          acc[i][r] = x;
        }
  }

  if (qi >= a.Sq) return;  // past the last row
  if (!live) {  // past the sample's: unmasked blocks have computed something for it
    l = 0.f;
#pragma unroll
    for (int i = 0; i < OB; ++i) acc[i] = gq_zero();
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no key seen: o = 0; NaN stays NaN
  const float lse = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
  T* orow = static_cast<T*>(a.out) + ((long long)it.b * a.Sq + qi) * a.ldo + (long long)head * a.dv;
  float* prow = a.part0 + ((((long long)it.split * a.B + it.b) * a.Sq + qi) * a.H + head) * a.dv;
#pragma unroll
  for (int i = 0; i < OB; ++i) {
    if (KW > 1 && i % KW != kw) continue;
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      const int d = 32 * i + 8 * g4 + 4 * h;
      if (d >= a.dv) continue;
      const float x[4] = {acc[i][4 * g4] * inv, acc[i][4 * g4 + 1] * inv, acc[i][4 * g4 + 2] * inv, acc[i][4 * g4 + 3] * inv};
      if (a.splits == 1) gq_store4(orow, d, a.dv, x);
      else gq_store4(prow, d, a.dv, x);
    }
  }
  if (h == 0 && kw == 0) {
    const long long at = ((long long)it.b * a.H + head) * a.Sq + qi;
    if (a.splits == 1) a.lse[at] = lse;
    else a.part1[(long long)it.split * a.B * a.H * a.Sq + at] = lse;
  }
}

// The parts of a row joined: 32 lanes a row of at most 128 columns. Each part is normalised, weight exp(lse_part - lse).
template <typename T>
__global__ __launch_bounds__(256) void gqa_fwd_join_kernel(GqaArgs a) {
  const long long rows = (long long)a.B * a.Sq * a.H, row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int d = 4 * (threadIdx.x & 31), head = (int)(row % a.H);
  const long long token = row / a.H, at = (token / a.Sq * a.H + head) * a.Sq + token % a.Sq;
  float top = -INFINITY;
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part1[s * rows + at]);
  float x[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
  if (top == -INFINITY) top = 0.f;  // no part saw a key
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float w = __builtin_amdgcn_exp2f((a.part1[s * rows + at] - top) * kLog2e);  // 0 of a part that saw none
    float v[4] = {};
    if (d < a.dv) load_piece(a.part0 + (s * rows + row) * a.dv, d, a.dv, v);
    sum += w;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = fmaf(w, v[i], x[i]);
  }
  if (d < a.dv) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] *= inv;
    gq_store4(static_cast<T*>(a.out) + token * a.ldo + (long long)head * a.dv, d, a.dv, x);
  }
  if (d == 0) a.lse[at] = sum == 0.f ? -INFINITY : top + logf(sum);
}

template <typename T>
__global__ __launch_bounds__(256) void gqa_join_kernel(int parts, size_t rows, int cols, const float* __restrict__ part,
                                                       T* __restrict__ out, long long ld) {
  const int per = (cols + 3) / 4;
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, row = i / per, n = rows * (size_t)cols;
  if (row >= rows) return;
  const int c = 4 * (int)(i % per);
  float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = 0; p < parts; ++p) {
    float v[4];
    load_piece(part + p * n + row * cols, c, cols, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] += v[j];
  }
  gq_store4(out + row * ld, c, cols, x);
}

template <typename T, int D, int NK, int KW, int NBUF, bool DMA = false>
int fwd_launch(GqaArgs a, hipStream_t s) {
  using S = FwdShape<T, D, NK, KW, NBUF>;
  const void* fn = a.bias ? (const void*)gqa_fwd_kernel<T, D, NK, KW, NBUF, true, DMA>
                          : (const void*)gqa_fwd_kernel<T, D, NK, KW, NBUF, false, DMA>;
  if (S::lds > 65536) TALOS_HIP(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)S::lds));
  const long long rows = (long long)a.G * a.Sq;
  a.tiles = (int)((rows + S::ROWS - 1) / S::ROWS);
  const long long base = (long long)a.tiles * a.B * a.KV;
  // Parts of the key loop, of at least 128 keys (4 samples' tokens against 512 keys: 13 us, 16 with 256), where there are fewer workgroups than the device holds: two a compute
  // unit, or one of the kernels that need a SIMD's registers for a wave. One token's workgroups of samples of different
  // lengths end at different times: twice as many there (64 samples of up to 4096 keys, 32 heads on 8, d 128: 130 us in
  // one part, 122 with the join in two, 122 in four).
  const long long fill = (KW > 1 && a.klens ? 1024 : 512) / (kFwdWaves<T, D> == 1 ? 2 : 1);
  long long splits = base >= fill ? 1 : (fill + base - 1) / base;
  splits = std::max(1ll, std::min(splits, ((long long)a.Sk + 127) / 128));
  TALOS_REQUIRE(base * splits <= 0x7fffffffll, TALOS_ERR_UNSUPPORTED, "talos_gqa_fwd: %lld workgroups", base * splits);
  a.splits = (int)splits;
  const size_t out_rows = (size_t)a.B * a.Sq * a.H;
  EntryScratch ws;
  int rc = ws.acquire(splits > 1 ? splits * out_rows * (a.dv + 1) * sizeof(float) : 0, s);
  if (rc) return rc;
  if (splits > 1) {
    a.part0 = static_cast<float*>(ws.ptr);
    a.part1 = a.part0 + splits * out_rows * a.dv;
  }
  void* args[] = {&a};
  rc = hip_status(hipLaunchKernel(fn, dim3((unsigned)(base * splits)), dim3(256), args, S::lds, s), "gqa_fwd_kernel");
  if (!rc && splits > 1) {
    hipLaunchKernelGGL(gqa_fwd_join_kernel<T>, dim3(ceil_div(out_rows, 8)), dim3(256), 0, s, a);
    rc = launch_status("gqa_fwd_join_kernel");
  }
  const int rel = ws.release();
  return rc ? rc : rel;
}

template <typename T>
int fwd(const char* fn, const talos_gqa_cfg* cfg, const int32_t* q_lens, const int32_t* k_lens, const float* bias,
        const T* q, long long ld_q, const T* k, long long ld_k, const T* v, long long ld_v, T* o, long long ld_o,
        float* lse, hipStream_t s) {
  int rc = gqa_check(fn, cfg, bias, q, ld_q, k, ld_k, v, ld_v, o, ld_o, lse);
  if (rc) return rc;
  TALOS_DEVICE();
  if (cfg->batch == 0 || cfg->q_len == 0) return entry_done(TALOS_OK, s);
  GqaArgs a = gqa_args(cfg, q_lens, k_lens, bias, q, ld_q, k, ld_k, v, ld_v);
  a.out = o;
  a.ldo = ld_o;
  a.lse = lse;
  const int d = std::max(a.dk, a.dv);
  // One wave's rows: the waves split the keys (64 samples' tokens against up to 4096 keys, d 128: 120 us, 184 where three
  // waves idle).
  const bool few = (long long)a.G * a.Sq <= 32;
  // Tiles of 64 bf16 keys, or 32 where direct and 128 wide (64: the same time) and of fp32, whose three planes leave no
  // room for more beside a second workgroup's. Direct tiles (gq_dma_fits) save the registers and the LDS stores: the decoding above 120 us, through registers 126; the
  // training that the backward is measured at 1627, 2260.
  if constexpr (sizeof(T) == 2) {
    const bool dma = a.dk == d && a.dv == d && gq_dma_fits(k, ld_k) && gq_dma_fits(v, ld_v);
    if (dma && d == 32) rc = few ? fwd_launch<T, 32, 32, 4, 1, true>(a, s) : fwd_launch<T, 32, 64, 1, 2, true>(a, s);
    else if (dma && d == 64) rc = few ? fwd_launch<T, 64, 32, 4, 1, true>(a, s) : fwd_launch<T, 64, 64, 1, 2, true>(a, s);
    else if (dma && d == 128) rc = few ? fwd_launch<T, 128, 32, 4, 1, true>(a, s) : fwd_launch<T, 128, 32, 1, 2, true>(a, s);
    else if (d <= 32) rc = few ? fwd_launch<T, 32, 32, 4, 1>(a, s) : fwd_launch<T, 32, 64, 1, 2>(a, s);
    else if (d <= 64) rc = few ? fwd_launch<T, 64, 32, 4, 1>(a, s) : fwd_launch<T, 64, 64, 1, 2>(a, s);
    else rc = few ? fwd_launch<T, 128, 32, 4, 1>(a, s) : fwd_launch<T, 128, 64, 1, 2>(a, s);
  } else {
    if (d <= 32) rc = few ? fwd_launch<T, 32, 32, 4, 1>(a, s) : fwd_launch<T, 32, 32, 1, 2>(a, s);
    else if (d <= 64) rc = few ? fwd_launch<T, 64, 32, 4, 1>(a, s) : fwd_launch<T, 64, 32, 1, 2>(a, s);
    else rc = few ? fwd_launch<T, 128, 32, 2, 1>(a, s) : fwd_launch<T, 128, 32, 1, 2>(a, s);
  }
  return entry_done(rc, s);
}

}  // namespace

template <typename T>
int gqa_join_launch(int parts, size_t rows, int cols, const float* part, T* out, long long ld, hipStream_t s) {
  const size_t n = rows * ((cols + 3) / 4);
  if (n == 0) return TALOS_OK;
  hipLaunchKernelGGL(gqa_join_kernel<T>, dim3(ceil_div(n, 256)), dim3(256), 0, s, parts, rows, cols, part, out, ld);
  return launch_status("gqa_join_kernel");
}
template int gqa_join_launch<float>(int, size_t, int, const float*, float*, long long, hipStream_t);
template int gqa_join_launch<Bf16>(int, size_t, int, const float*, Bf16*, long long, hipStream_t);

int gqa_check(const char* fn, const talos_gqa_cfg* cfg, const float* bias, const void* q, long long ld_q, const void* k,
              long long ld_k, const void* v, long long ld_v, const void* o, long long ld_o, const float* lse) {
  TALOS_REQUIRE(cfg != nullptr, TALOS_ERR_NULL, "%s: null configuration", fn);
  const talos_gqa_cfg& c = *cfg;
  TALOS_REQUIRE(c.batch >= 0 && c.q_len >= 0 && c.k_len >= 0 && c.heads > 0 && c.kv_heads > 0 && c.qk_dim > 0 &&
                    c.v_dim > 0,
                TALOS_ERR_SHAPE, "%s: bad shape (batch=%d q_len=%d k_len=%d heads=%d kv_heads=%d qk_dim=%d v_dim=%d)", fn,
                c.batch, c.q_len, c.k_len, c.heads, c.kv_heads, c.qk_dim, c.v_dim);
  TALOS_REQUIRE(c.heads % c.kv_heads == 0, TALOS_ERR_SHAPE, "%s: %d heads do not divide into %d groups", fn, c.heads,
                c.kv_heads);
  TALOS_REQUIRE(c.qk_dim <= 128 && c.v_dim <= 128, TALOS_ERR_UNSUPPORTED, "%s: head dims (%d, %d) exceed 128", fn,
                c.qk_dim, c.v_dim);
  TALOS_REQUIRE(c.causal == 0 || c.causal == 1, TALOS_ERR_DTYPE, "%s: causal must be 0 or 1", fn);
  TALOS_REQUIRE(c.scale > 0.f && c.scale < INFINITY, TALOS_ERR_SHAPE, "%s: scale must be positive and finite", fn);
  TALOS_REQUIRE(c.scale >= 1e-30f && c.scale <= 1e30f, TALOS_ERR_UNSUPPORTED, "%s: scale %g is not within 1e-30 .. 1e30",
                fn, (double)c.scale);
  TALOS_REQUIRE(!bias || (c.max_distance > 0 && c.max_distance <= (1 << 20)), TALOS_ERR_SHAPE,
                "%s: a bias needs 1 <= max_distance <= 2^20, not %d", fn, c.max_distance);
  // rows of a sample's group and keys are counted in 32 bits (with a tile's length of room), addresses in 64
  TALOS_REQUIRE((long long)c.q_len * c.heads <= (1 << 30) && c.k_len <= (1 << 30) &&
                    (long long)c.batch * c.heads <= (1 << 30),
                TALOS_ERR_UNSUPPORTED, "%s: q_len * heads, k_len or batch * heads exceeds 2^30", fn);
  TALOS_REQUIRE(ld_q >= (long long)c.heads * c.qk_dim && ld_k >= (long long)c.kv_heads * c.qk_dim &&
                    ld_v >= (long long)c.kv_heads * c.v_dim && ld_o >= (long long)c.heads * c.v_dim,
                TALOS_ERR_SHAPE, "%s: a row stride is smaller than heads * dim", fn);
  const bool queries = c.batch > 0 && c.q_len > 0, keys = c.batch > 0 && c.k_len > 0;
  TALOS_REQUIRE((!queries || (q && o && lse)) && (!keys || (k && v)), TALOS_ERR_NULL, "%s: null q, k, v, o or lse", fn);
  return TALOS_OK;
}

GqaArgs gqa_args(const talos_gqa_cfg* cfg, const int32_t* q_lens, const int32_t* k_lens, const float* bias, const void* q,
                 long long ld_q, const void* k, long long ld_k, const void* v, long long ld_v) {
  GqaArgs a{};
  a.B = cfg->batch;
  a.Sq = cfg->q_len;
  a.Sk = cfg->k_len;
  a.H = cfg->heads;
  a.KV = cfg->kv_heads;
  a.G = cfg->heads / cfg->kv_heads;
  a.dk = cfg->qk_dim;
  a.dv = cfg->v_dim;
  a.causal = cfg->causal;
  a.M = bias ? cfg->max_distance : 0;
  a.scale = cfg->scale;
  a.c = cfg->scale * kLog2e;
  a.qlens = q_lens;
  a.klens = k_lens;
  a.bias = bias;
  a.q = q;
  a.k = k;
  a.v = v;
  a.ldq = ld_q;
  a.ldk = ld_k;
  a.ldv = ld_v;
  return a;
}

}  // namespace talos

using namespace talos;

extern "C" {

int talos_gqa_fwd_f32(const talos_gqa_cfg* cfg, const int32_t* q_lens, const int32_t* k_lens, const float* bias,
                      const float* q, long long ld_q, const float* k, long long ld_k, const float* v, long long ld_v,
                      float* o, long long ld_o, float* lse, talos_stream_t stream) {
  return fwd<float>(__func__, cfg, q_lens, k_lens, bias, q, ld_q, k, ld_k, v, ld_v, o, ld_o, lse, as_stream(stream));
}
int talos_gqa_fwd_bf16(const talos_gqa_cfg* cfg, const int32_t* q_lens, const int32_t* k_lens, const float* bias,
                       const talos_bf16* q, long long ld_q, const talos_bf16* k, long long ld_k, const talos_bf16* v,
                       long long ld_v, talos_bf16* o, long long ld_o, float* lse, talos_stream_t stream) {
  return fwd<Bf16>(__func__, cfg, q_lens, k_lens, bias, reinterpret_cast<const Bf16*>(q), ld_q,
                   reinterpret_cast<const Bf16*>(k), ld_k, reinterpret_cast<const Bf16*>(v), ld_v,
                   reinterpret_cast<Bf16*>(o), ld_o, lse, as_stream(stream));
}

}  // extern "C"
