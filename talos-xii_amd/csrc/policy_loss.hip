// policy_loss.hip -- the clipped policy loss with a KL term from wide rows of logits, and its gradient.
//
// Row t holds the logits x of one decision or token, of which action a was taken:
//   logp = x_a - log sum_j exp(x_j),   ratio = exp(logp - old_logp)
//   gain = min(ratio adv, clip(ratio, 1 - low, 1 + high) adv)
//   kl   = exp(ref_logp - logp) - (ref_logp - logp) - 1
//   loss = sum_t weight_t (kl_coef kl_t - gain_t)
//   dloss / dx_j = slope (1[j = a] - p_j),  slope = weight (kl_coef (1 - exp(ref_logp - logp)) - adv ratio 1[not clipped])
// (src/ppo.rs:702-749 has the loss per sample over five actions; the reference has no KL term.)
//
// Bound by memory: a row is read once into registers (as its raw 16-byte pieces, so bf16 rows take half
// the registers), its maximum, its sum of exponentials and the taken logit are formed, and the gradient
// is written from the same registers: one read and one write of the logits for loss and gradient
// together. L lanes hold a row, V pieces each: 8 lanes up to 32 (fp32) or 64 (bf16) actions, a wave
// up to 2048 or 4096, four waves or eight beyond, up to 32768 columns; wider rows are read again. The
// exponentials are fp32 (f64 in rows of a few values), their sums f64 from a piece on.
//
// Rows of weight 0 are padding: their logits are not read, their gradient is zero.
#include <algorithm>
#include <cmath>

#include "vecio.hpp"

namespace talos {

namespace {

// partial sums of a workgroup: the loss, then the entries of enum talos_policy_stat
constexpr int kPolParts = 1 + TALOS_POLICY_NSTATS;
// 16-byte pieces of a row that eight waves hold, 8 or (fp32) 16 a lane; a wider row is read again, from cache. Eight waves
// leave room for other rows at other phases: 4096 x 20001 bf16 97 us, with sixteen of half the pieces 109; 4096 x 32768 115
// and 117, reading again 136. 16 a lane hold fp32 rows of twice as many pieces (2048 x 30001 110 us, 134 reading again; x
// 20000 75 and 85); of bf16 rows, twice as many values, they gain near the full width alone (x 60000 126 and 136, x 40000
// 95 and 89).
template <typename T>
constexpr int kHeld = sizeof(T) == 4 ? 8192 : 4096;
constexpr int kPolicyMaxVocab = 1 << 26;

struct PolicyArgs {
  int rows, vocab;
  float clip_low, clip_high, kl_coef;
  double log_low, log_high, even;  // of the clip's borders; the weight of a row where all count alike
  long long ld, ld_d;
  const int32_t* actions;
  const float *adv, *old_logp, *ref_logp, *weight;
  float* logp;
  double* part;  // [gridDim.x][kPolParts], or null
};

// What a row's loss and gradient need of it.
struct RowTerms {
  double sums[kPolParts];
  float slope, logp;
};

// A row's scalars are f64: gains of either sign cancel in the loss (to a hundredth of their size over a minibatch), and
// so do ratio - 1 and its logarithm. The library's f64 exp, expm1 and log cost 400 instructions a row between them, a third of
// the time of rows of 3000 bf16 values; these are a fifth of it, to 2^-41 (8192 x 2999 bf16: 32.4 us, with fp32 functions
// and sums 30.1, whose loss was 10 to 100 times less exact; 4096 x 32768 bf16 117 us, 115).
struct Exp {
  double value, less, rest;  // exp(d), exp(d) - 1, exp(d) - 1 - d
};
// 2^n exp(r) with |r| <= ln 2 / 2, exp(r) = 1 + r + r^2 (1/2 + r/6 + ... + r^8/10!): the next term is below 2^-42
__device__ __forceinline__ Exp exp_f64(double d) {
  const double held = fmin(fmax(d, -2000.0), 2000.0);
  const double n = rint(held * 1.4426950408889634);
  // ln 2 in two parts, the first of 31 bits, so that n times it is exact
  constexpr double kHi = 1488522236.0 / 2147483648.0, kLo = -4.2009150726810846e-11;
  const double r = fma(n, -kLo, fma(n, -kHi, held));
  double q = 1.0 / 3628800.0;
  q = fma(q, r, 1.0 / 362880.0);
  q = fma(q, r, 1.0 / 40320.0);
  q = fma(q, r, 1.0 / 5040.0);
  q = fma(q, r, 1.0 / 720.0);
  q = fma(q, r, 1.0 / 120.0);
  q = fma(q, r, 1.0 / 24.0);
  q = fma(q, r, 1.0 / 6.0);
  q = fma(q, r, 0.5);
  q = q * r * r;
  Exp e;
  e.value = d != d ? d : ldexp(q + r + 1.0, (int)n);
  e.less = n == 0.0 ? q + r : e.value - 1.0;
  e.rest = n == 0.0 ? q : e.less - d;
  return e;
}
// log z = n ln 2 + 2 atanh((m - 1) / (m + 1)), m within sqrt(1/2) .. sqrt(2): the term left out is below 2^-44
__device__ __forceinline__ double log_f64(double z) {
  int n;
  double m = frexp(z, &n);
  if (m < 0.70710678118654752) {
    m += m;
    --n;
  }
  const double s = (m - 1.0) / (m + 1.0), t = s * s;
  double p = 2.0 / 15.0;
  p = fma(p, t, 2.0 / 13.0);
  p = fma(p, t, 2.0 / 11.0);
  p = fma(p, t, 2.0 / 9.0);
  p = fma(p, t, 2.0 / 7.0);
  p = fma(p, t, 2.0 / 5.0);
  p = fma(p, t, 2.0 / 3.0);
  p = fma(p, t, 2.0);
  return fma((double)n, 0.69314718055994531, p * s);
}

// From the row's maximum, the sum of its exponentials and the taken logit. An action out of range has no
// log-probability: a NaN loss and no gradient.
__device__ __forceinline__ RowTerms policy_row(const PolicyArgs& a, int row, bool bad, float top, double sum,
                                               float taken) {
  RowTerms t;
  const double w = a.weight ? (double)a.weight[row] : a.even;
  const double logp = bad ? (double)NAN : ((double)taken - (double)top) - log_f64(sum);
  const double adv = a.adv[row], diff = logp - (double)a.old_logp[row];
  const Exp ratio = exp_f64(diff);
  const bool up = adv >= 0.0, clipped = up ? diff > a.log_high : diff < a.log_low;
  // the smaller of ratio adv and the clipped ratio's
  const double gain = adv * (clipped ? (up ? 1.0 + (double)a.clip_high : 1.0 - (double)a.clip_low) : ratio.value);
  double kl = 0.0, dkl = 0.0;
  if (a.ref_logp) {
    const double gap = (double)a.ref_logp[row] - logp;
    const Exp e = exp_f64(gap);
    kl = e.rest;
    dkl = -e.less;
  }
  t.sums[0] = bad ? (double)NAN : w * ((double)a.kl_coef * kl - gain);
  t.sums[1 + TALOS_POLICY_STAT_KL] = ratio.rest;  // (ratio - 1) - log ratio
  t.sums[1 + TALOS_POLICY_STAT_POLICY] = gain;
  t.sums[1 + TALOS_POLICY_STAT_REF_KL] = kl;
  t.sums[1 + TALOS_POLICY_STAT_CLIPPED] = clipped ? 1.0 : 0.0;
  t.sums[1 + TALOS_POLICY_STAT_COUNT] = 1.0;
  t.slope = bad ? 0.f : (float)(w * ((double)a.kl_coef * dkl - (clipped ? 0.0 : adv * ratio.value)));
  t.logp = (float)logp;
  return t;
}

// The exponentials of a piece's values less the row's maximum, added up: fp32 ones and sums of a piece, as their roundings
// average out over a long row (that of log2(e) itself, 1.3e-8 of every exponent, does not, and is put right); f64 ones in
// rows of a few values (EXACT), where they do not.
constexpr float kLog2e = 1.44269504f, kLog2eRest = (float)(1.4426950408889634 - (double)kLog2e);
template <bool EXACT, int N>
__device__ __forceinline__ double exp_sum(const float (&v)[N], float top) {
  if constexpr (EXACT) {
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) s += exp_f64((double)v[i] - (double)top).value;
    return s;
  } else {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float x = v[i] - top;
      s += __builtin_amdgcn_exp2f(fmaf(x, kLog2e, x * kLog2eRest));
    }
    return (double)s;
  }
}
__device__ __forceinline__ double lanes_sum_f64(double v, int lanes) {
  for (int o = lanes / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

// What a value adds to the sum of a lane or wave that has no maximum (every value -inf, or NaN): a NaN still shows.
__device__ __forceinline__ float none_or_nan(float v) { return v == -INFINITY ? 0.f : v; }

// One row per L lanes. V > 0: the row stays in registers, V pieces a lane; V = 0: any width, read again for the gradient
// (L = 1024). dlogits null: the loss alone. dlogits may be the logits' own rows. (A workgroup that walks several rows
// with the next one in flight holds the f64 constants over the loop, one workgroup a compute unit for two: 131 -> 160 us
// at 4096 x 32768 bf16.)
template <typename T, int L, int V>
__global__ __launch_bounds__(L > 256 ? L : 256) void policy_loss_kernel(PolicyArgs a, const T* logits, T* dlogits) {
  constexpr int N = Piece<T>::N, TB = L > 256 ? L : 256, R = TB / L, W = L > 64 ? L / 64 : 1;
  constexpr int LW = L < 64 ? L : 64;
  __shared__ float tops[W], slope_of[1];
  __shared__ double sums[W];
  __shared__ double part[R][kPolParts];
  const int lane = threadIdx.x % L, sub = threadIdx.x / L;
  const long long row = (long long)blockIdx.x * R + sub;
  const bool in = row < a.rows;
  const bool on = in && (!a.weight || a.weight[row] != 0.f);  // W > 1: one answer for the workgroup
  const T* xr = logits + (in ? row : 0) * a.ld;
  T* dr = dlogits ? dlogits + (in ? row : 0) * a.ld_d : nullptr;
  if (lane < kPolParts) part[sub][lane] = 0.0;
  float top = -INFINITY, slope = 0.f;
  double sum = 0.0;
  int act = -1;
  typename Piece<T>::Raw raw[V ? V : 1];
  if (on) {
    act = a.actions[row];
    const float taken = act < 0 || act >= a.vocab ? 0.f : to_f32(xr[act]);
    if constexpr (V > 0) {
      // values past the row are -inf: no maximum, no share of the sum
#pragma unroll
      for (int j = 0; j < V; ++j) raw[j] = row_piece(xr, N * (lane + L * j), a.vocab, -INFINITY);
#pragma unroll
      for (int j = 0; j < V; ++j) row_piece_end<T>(raw[j], N * (lane + L * j), a.vocab, -INFINITY);
      auto each = [&](auto&& f) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float v[N];
          // opaque to the compiler, which would otherwise widen the row once and hold it so (232 spills)
#pragma unroll
          for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(raw[j].w[i]));
          Piece<T>::widen(raw[j], v);
          f(v);
        }
      };
      each([&](const float(&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) top = fmaxf(top, v[i]);
      });
      top = lanes_max<LW>(top);
      if (top > -INFINITY) {
        each([&](const float(&v)[N]) { sum += exp_sum<(L < 64)>(v, top); });
      } else {
        each([&](const float(&v)[N]) {
#pragma unroll
          for (int i = 0; i < N; ++i) sum += (double)none_or_nan(v[i]);
        });
      }
    } else {
      // one pass with each lane's running maximum, U pieces at a time
      constexpr int U = 2;
      for (int c0 = N * lane; c0 < a.vocab; c0 += U * N * L) {
        float v[U][N], most = top;
#pragma unroll
        for (int u = 0; u < U; ++u) load_piece(xr, c0 + u * N * L, a.vocab, v[u], -INFINITY);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < N; ++i) most = fmaxf(most, v[u][i]);
        if (most > -INFINITY) {
          if (most > top) sum *= exp_f64((double)top - (double)most).value;
#pragma unroll
          for (int u = 0; u < U; ++u) sum += exp_sum<false>(v[u], most);
          top = most;
        } else {
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < N; ++i) sum += (double)none_or_nan(v[u][i]);
        }
      }
      const float mine = top;
      top = lanes_max<LW>(top);
      sum *= mine == -INFINITY ? 1.0 : exp_f64((double)mine - (double)top).value;
    }
    sum = lanes_sum_f64(sum, LW);
    if constexpr (W > 1) {
      // the waves' maxima and sums, joined by every wave
      if ((threadIdx.x & 63) == 0) {
        tops[threadIdx.x >> 6] = top;
        sums[threadIdx.x >> 6] = sum;
      }
      __syncthreads();
      const int l64 = threadIdx.x & 63;
      const float its = l64 < W ? tops[l64] : -INFINITY;
      top = lanes_max<W>(its);
      top = __shfl(top, 0, kWave);
      sum = lanes_sum_f64(l64 < W ? sums[l64] * (its == -INFINITY ? 1.0 : exp_f64((double)its - (double)top).value) : 0.0, W);
      sum = __shfl(sum, 0, kWave);
    }
    if (top == -INFINITY) sum = (double)NAN;  // no maximum in the whole row: no distribution
    // the row's scalars: one wave's work, not every wave's
    if (W == 1 || threadIdx.x < 64) {
      const RowTerms t = policy_row(a, (int)row, act < 0 || act >= a.vocab, top, sum, taken);
      slope = t.slope;
      if (lane == 0) {
        if (a.logp) a.logp[row] = t.logp;
        if (W > 1) slope_of[0] = t.slope;
#pragma unroll
        for (int i = 0; i < kPolParts; ++i) part[sub][i] = t.sums[i];
      }
    }
    if constexpr (W > 1) {
      __syncthreads();
      slope = slope_of[0];
    }
  } else if (in && lane == 0 && a.logp) {
    a.logp[row] = 0.f;
  }
  if (a.part) {
    __syncthreads();
    if (threadIdx.x < kPolParts) {
      double s = 0.0;
      for (int r = 0; r < R; ++r) s += part[r][threadIdx.x];
      a.part[(size_t)blockIdx.x * kPolParts + threadIdx.x] = s;
    }
  }
  if (!in || !dr) return;
  const float scale = -slope / (float)sum;
  auto grad = [&](float (&v)[N], int c) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = on ? __expf(v[i] - top) * scale : 0.f;
      if (on && c + i == act) v[i] += slope;
    }
    store_piece(dr, c, a.vocab, v);
  };
  if constexpr (V > 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = N * (lane + L * j);
      if (c >= a.vocab) continue;
      float v[N];
      Piece<T>::widen(raw[j], v);
      grad(v, c);
    }
  } else {
    constexpr int U = 2;
    for (int c0 = N * lane; c0 < a.vocab; c0 += U * N * L) {
      float v[U][N] = {};
      if (on)
#pragma unroll
        for (int u = 0; u < U; ++u) load_piece(xr, c0 + u * N * L, a.vocab, v[u]);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + u * N * L < a.vocab) grad(v[u], c0 + u * N * L);
    }
  }
}

// The partial rows' sums in a fixed order: thread t every 1024th row, then the waves' trees. (A wave a quantity took 20 us
// over 4096 rows, waiting for 64 loads in turn.)
__global__ __launch_bounds__(1024) void policy_loss_final_kernel(int nblk, const double* __restrict__ part,
                                                                 float* __restrict__ loss, double* stats, int accumulate) {
  __shared__ double red[16][kPolParts];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  double s[kPolParts] = {};
#pragma unroll 4
  for (int k = threadIdx.x; k < nblk; k += 1024)
#pragma unroll
    for (int i = 0; i < kPolParts; ++i) s[i] += part[(size_t)k * kPolParts + i];
#pragma unroll
  for (int i = 0; i < kPolParts; ++i) {
    s[i] = wave_sum(s[i]);
    if (lane == 0) red[wv][i] = s[i];
  }
  __syncthreads();
  const int i = threadIdx.x;
  if (i >= kPolParts) return;
  double t = 0.0;
#pragma unroll
  for (int w = 0; w < 16; ++w) t += red[w][i];
  if (i == 0) {
    if (loss) loss[0] = (float)t;
  } else if (stats) {
    stats[i - 1] = (accumulate ? stats[i - 1] : 0.0) + t;
  }
}

template <typename T>
int policy_loss(const char* fn, int rows, int vocab, float clip_low, float clip_high, float kl_coef, const T* logits,
                long long ld, const int32_t* actions, const float* adv, const float* old_logp, const float* ref_logp,
                const float* weight, T* dlogits, long long ld_d, float* loss, float* logp, double* stats,
                int accumulate, hipStream_t s) {
  TALOS_REQUIRE(rows >= 0 && vocab > 0, TALOS_ERR_SHAPE, "%s: bad shape rows=%d vocab=%d", fn, rows, vocab);
  TALOS_REQUIRE(vocab <= kPolicyMaxVocab, TALOS_ERR_UNSUPPORTED, "%s: vocab %d exceeds %d", fn, vocab, kPolicyMaxVocab);
  TALOS_REQUIRE(clip_low >= 0.f && clip_high >= 0.f, TALOS_ERR_SHAPE, "%s: clip_low and clip_high must be >= 0", fn);
  TALOS_REQUIRE(ld >= vocab && (!dlogits || ld_d >= vocab), TALOS_ERR_SHAPE, "%s: a row stride is smaller than vocab",
                fn);
  TALOS_REQUIRE(!dlogits || (const void*)dlogits != (const void*)logits || ld == ld_d, TALOS_ERR_SHAPE,
                "%s: dlogits in the logits' place needs their row stride", fn);
  TALOS_REQUIRE(accumulate == 0 || accumulate == 1, TALOS_ERR_SHAPE, "%s: stats_accumulate must be 0 or 1", fn);
  TALOS_REQUIRE(rows == 0 || (logits && actions && adv && old_logp), TALOS_ERR_NULL, "%s: null input", fn);
  TALOS_REQUIRE(kl_coef == 0.f || ref_logp || rows == 0, TALOS_ERR_NULL, "%s: kl_coef without ref_logp", fn);
  TALOS_DEVICE();
  constexpr int N = Piece<T>::N;
  const int pieces = (vocab + N - 1) / N;
  PolicyArgs a{rows, vocab, clip_low, clip_high, kl_coef, std::log(std::max(0.0, 1.0 - (double)clip_low)),
               std::log1p((double)clip_high), rows ? 1.0 / (double)rows : 0.0, ld, ld_d, actions, adv, old_logp,
               ref_logp, weight, logp, nullptr};
  const int per = pieces <= 8 ? 32 : pieces <= 512 ? 4 : 1;  // rows a workgroup
  const int nblk = (int)ceil_div((size_t)rows, per);
  EntryScratch ws;
  int rc = ws.acquire(loss || stats ? (size_t)nblk * kPolParts * sizeof(double) : 0, s);
  if (rc) return rc;
  a.part = static_cast<double*>(ws.ptr);
  if (nblk > 0) {
#define TALOS_POL(L, V)                                                                                          \
  hipLaunchKernelGGL((policy_loss_kernel<T, L, V>), dim3(nblk), dim3(L > 256 ? L : 256), 0, s, a, logits, dlogits)
    if (pieces > kHeld<T>) TALOS_POL(1024, 0);
    else if (pieces <= 8) TALOS_POL(8, 1);
    else if (pieces <= 64) TALOS_POL(64, 1);
    else if (pieces <= 256) TALOS_POL(64, 4);
    else if (pieces <= 512) TALOS_POL(64, 8);
    else if (pieces <= 1024) TALOS_POL(256, 4);
    else if (pieces <= 2048) TALOS_POL(256, 8);
    else if (pieces <= 4096) TALOS_POL(512, 8);
    else if constexpr (sizeof(T) == 4) TALOS_POL(512, 16);
#undef TALOS_POL
    rc = launch_status("policy_loss_kernel");
  }
  if (!rc && (loss || stats)) {
    hipLaunchKernelGGL(policy_loss_final_kernel, dim3(1), dim3(1024), 0, s, nblk, a.part, loss, stats,
                       accumulate);
    rc = launch_status("policy_loss_final_kernel");
  }
  const int rel = ws.release();
  return entry_done(rc ? rc : rel, s);
}

}  // namespace
}  // namespace talos

using namespace talos;

extern "C" {

int talos_policy_loss_fwd_f32(int rows, int vocab, float clip_low, float clip_high, float kl_coef, const float* logits,
                              long long ld_logits, const int32_t* actions, const float* adv, const float* old_logp,
                              const float* ref_logp, const float* weight, float* loss, float* logp, double* stats,
                              int stats_accumulate, talos_stream_t stream) {
  TALOS_REQUIRE(loss || logp || stats, TALOS_ERR_NULL, "%s: loss, logp and stats are all null", __func__);
  return policy_loss<float>(__func__, rows, vocab, clip_low, clip_high, kl_coef, logits, ld_logits, actions, adv,
                            old_logp, ref_logp, weight, nullptr, 0, loss, logp, stats, stats_accumulate,
                            as_stream(stream));
}
int talos_policy_loss_fwd_bf16(int rows, int vocab, float clip_low, float clip_high, float kl_coef,
                               const talos_bf16* logits, long long ld_logits, const int32_t* actions, const float* adv,
                               const float* old_logp, const float* ref_logp, const float* weight, float* loss,
                               float* logp, double* stats, int stats_accumulate, talos_stream_t stream) {
  TALOS_REQUIRE(loss || logp || stats, TALOS_ERR_NULL, "%s: loss, logp and stats are all null", __func__);
  return policy_loss<Bf16>(__func__, rows, vocab, clip_low, clip_high, kl_coef, reinterpret_cast<const Bf16*>(logits),
                           ld_logits, actions, adv, old_logp, ref_logp, weight, nullptr, 0, loss, logp, stats,
                           stats_accumulate, as_stream(stream));
}
int talos_policy_loss_bwd_f32(int rows, int vocab, float clip_low, float clip_high, float kl_coef, const float* logits,
                              long long ld_logits, const int32_t* actions, const float* adv, const float* old_logp,
                              const float* ref_logp, const float* weight, float* dlogits, long long ld_dlogits,
                              float* loss, float* logp, double* stats, int stats_accumulate, talos_stream_t stream) {
  TALOS_REQUIRE(dlogits || rows == 0, TALOS_ERR_NULL, "%s: null pointer argument 'dlogits'", __func__);
  return policy_loss<float>(__func__, rows, vocab, clip_low, clip_high, kl_coef, logits, ld_logits, actions, adv,
                            old_logp, ref_logp, weight, dlogits, ld_dlogits, loss, logp, stats, stats_accumulate,
                            as_stream(stream));
}
int talos_policy_loss_bwd_bf16(int rows, int vocab, float clip_low, float clip_high, float kl_coef,
                               const talos_bf16* logits, long long ld_logits, const int32_t* actions, const float* adv,
                               const float* old_logp, const float* ref_logp, const float* weight, talos_bf16* dlogits,
                               long long ld_dlogits, float* loss, float* logp, double* stats, int stats_accumulate,
                               talos_stream_t stream) {
  TALOS_REQUIRE(dlogits || rows == 0, TALOS_ERR_NULL, "%s: null pointer argument 'dlogits'", __func__);
  return policy_loss<Bf16>(__func__, rows, vocab, clip_low, clip_high, kl_coef, reinterpret_cast<const Bf16*>(logits),
                           ld_logits, actions, adv, old_logp, ref_logp, weight, reinterpret_cast<Bf16*>(dlogits),
                           ld_dlogits, loss, logp, stats, stats_accumulate, as_stream(stream));
}

}  // extern "C"
