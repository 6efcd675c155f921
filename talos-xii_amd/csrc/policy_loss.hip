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
// up to 2048 or 4096, four waves or sixteen beyond, up to 16384 fp32 or 32768 bf16 columns; wider rows are read again. The sums
// are fp32 (at most a few dozen terms a lane, then a tree).
//
// Rows of weight 0 are padding: their logits are not read, their gradient is zero.
#include <algorithm>
#include <cmath>

#include "vecio.hpp"

namespace talos {

namespace {

// partial sums of a workgroup: the loss, then the entries of enum talos_policy_stat
constexpr int kPolParts = 1 + TALOS_POLICY_NSTATS;
// 16-byte pieces of a row that sixteen waves hold (4 a lane). With 8 a lane a compute unit no longer has room for two
// workgroups, and reading the row again, from cache, is faster: 2048 x 30001 fp32 138 -> 130 us, x 40000 bf16 114 -> 82;
// with 4, holding is: 4096 x 32768 bf16 136 -> 119 us.
constexpr int kHeld = 4096;
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

// exp(g) - g - 1: by its series near 0, where the difference would keep few digits
__device__ __forceinline__ float exp_rest(float g) {
  if (fabsf(g) < 0.25f) {
    // 1/2 + g (1/6 + g (1/24 + ...)), the term left out below 2^-25 of the first
    const float p = fmaf(g, fmaf(g, fmaf(g, fmaf(g, fmaf(g, 1.f / 5040.f, 1.f / 720.f), 1.f / 120.f), 1.f / 24.f), 1.f / 6.f), 0.5f);
    return g * g * p;
  }
  return expm1f(g) - g;
}

// From the row's maximum, the sum of its exponentials and the taken logit. An action out of range has no
// log-probability: a NaN loss and no gradient. Log-probabilities and their differences are f64, as the clip's border is
// looked up in them; the exponentials of the differences are fp32 (the f64 functions, 400 instructions a row and their
// constants, took a third of the time of rows of 3000 bf16 values).
__device__ __forceinline__ RowTerms policy_row(const PolicyArgs& a, int row, bool bad, float top, float sum,
                                               float taken) {
  RowTerms t;
  const double w = a.weight ? (double)a.weight[row] : a.even;
  int n;
  const float part = frexpf(sum, &n);  // log sum: to 2^-25, whatever its size
  const double logz = fma((double)n, 0.69314718055994531, (double)logf(part));
  const double logp = bad ? (double)NAN : ((double)taken - (double)top) - logz;
  const double adv = a.adv[row], diff = logp - (double)a.old_logp[row];
  const float ratio = expf((float)diff);
  const bool up = adv >= 0.0, clipped = up ? diff > a.log_high : diff < a.log_low;
  // the smaller of ratio adv and the clipped ratio's
  const double gain = adv * (clipped ? (up ? 1.0 + (double)a.clip_high : 1.0 - (double)a.clip_low) : (double)ratio);
  float kl = 0.f, dkl = 0.f;
  if (a.ref_logp) {
    const float gap = (float)((double)a.ref_logp[row] - logp);
    kl = exp_rest(gap);
    dkl = -expm1f(gap);
  }
  t.sums[0] = bad ? (double)NAN : w * ((double)a.kl_coef * kl - gain);
  t.sums[1 + TALOS_POLICY_STAT_KL] = exp_rest((float)diff);  // (ratio - 1) - log ratio
  t.sums[1 + TALOS_POLICY_STAT_POLICY] = gain;
  t.sums[1 + TALOS_POLICY_STAT_REF_KL] = kl;
  t.sums[1 + TALOS_POLICY_STAT_CLIPPED] = clipped ? 1.0 : 0.0;
  t.sums[1 + TALOS_POLICY_STAT_COUNT] = 1.0;
  t.slope = bad ? 0.f : (float)(w * ((double)a.kl_coef * dkl - (clipped ? 0.0 : adv * ratio)));
  t.logp = (float)logp;
  return t;
}

// What a value adds to the sum of a lane or wave that has no maximum (every value -inf, or NaN): a NaN still shows.
__device__ __forceinline__ float none_or_nan(float v) { return v == -INFINITY ? 0.f : v; }

// One row per L lanes. V > 0: the row stays in registers, V pieces a lane; V = 0: any width, read again for the gradient
// (L = 1024). dlogits null: the loss alone. dlogits may be the logits' own rows. (A workgroup that walks several rows
// with the next one in flight holds the f64 functions' constants over the loop: 128 registers for 28, one workgroup a
// compute unit for two, 131 -> 160 us at 4096 x 32768 bf16.)
template <typename T, int L, int V>
__global__ __launch_bounds__(L > 256 ? L : 256) void policy_loss_kernel(PolicyArgs a, const T* logits, T* dlogits) {
  constexpr int N = Piece<T>::N, TB = L > 256 ? L : 256, R = TB / L, W = L > 64 ? L / 64 : 1;
  constexpr int LW = L < 64 ? L : 64;
  __shared__ float tops[W], sums[W], slope_of[1];
  __shared__ double part[R][kPolParts];
  const int lane = threadIdx.x % L, sub = threadIdx.x / L;
  const long long row = (long long)blockIdx.x * R + sub;
  const bool in = row < a.rows;
  const bool on = in && (!a.weight || a.weight[row] != 0.f);  // W > 1: one answer for the workgroup
  const T* xr = logits + (in ? row : 0) * a.ld;
  T* dr = dlogits ? dlogits + (in ? row : 0) * a.ld_d : nullptr;
  if (lane < kPolParts) part[sub][lane] = 0.0;
  float top = -INFINITY, sum = 0.f, slope = 0.f;
  int act = -1;
  typename Piece<T>::Raw raw[V ? V : 1];
  if (on) {
    act = a.actions[row];
    const float taken = act < 0 || act >= a.vocab ? 0.f : to_f32(xr[act]);
    if constexpr (V > 0) {
      // values past the row are -inf: no maximum, no share of the sum
#pragma unroll
      for (int j = 0; j < V; ++j) raw[j] = load_raw(xr, N * (lane + L * j), a.vocab, -INFINITY);
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
        each([&](const float(&v)[N]) {
#pragma unroll
          for (int i = 0; i < N; ++i) sum += __expf(v[i] - top);
        });
      } else {
        each([&](const float(&v)[N]) {
#pragma unroll
          for (int i = 0; i < N; ++i) sum += none_or_nan(v[i]);
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
          sum *= __expf(top - most);
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < N; ++i) sum += __expf(v[u][i] - most);
          top = most;
        } else {
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < N; ++i) sum += none_or_nan(v[u][i]);
        }
      }
      const float mine = top;
      top = lanes_max<LW>(top);
      sum *= mine == -INFINITY ? 1.f : __expf(mine - top);
    }
    sum = lanes_sum<LW>(sum);
    if constexpr (W > 1) {
      // the waves' maxima and sums, joined by every wave
      if ((threadIdx.x & 63) == 0) {
        tops[threadIdx.x >> 6] = top;
        sums[threadIdx.x >> 6] = sum;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < W; ++i) top = fmaxf(top, tops[i]);
      sum = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) sum += sums[i] * (tops[i] == -INFINITY ? 1.f : __expf(tops[i] - top));
    }
    if (top == -INFINITY) sum = NAN;  // no maximum in the whole row: no distribution
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
  const float scale = -slope / sum;
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
               std::log1p((double)clip_high), rows ? 1.0 / (double)rows : 0.0, ld, ld_d, actions, adv, old_logp, ref_logp, weight, logp,
               nullptr};
  const int per = pieces <= 8 ? 32 : pieces <= 512 ? 4 : 1;  // rows a workgroup
  const int nblk = (int)ceil_div((size_t)rows, per);
  EntryScratch ws;
  int rc = ws.acquire(loss || stats ? (size_t)nblk * kPolParts * sizeof(double) : 0, s);
  if (rc) return rc;
  a.part = static_cast<double*>(ws.ptr);
  if (nblk > 0) {
#define TALOS_POL(L, V)                                                                                          \
  hipLaunchKernelGGL((policy_loss_kernel<T, L, V>), dim3(nblk), dim3(L > 256 ? L : 256), 0, s, a, logits, dlogits)
    if (pieces > kHeld) TALOS_POL(1024, 0);
    else if (pieces <= 8) TALOS_POL(8, 1);
    else if (pieces <= 64) TALOS_POL(64, 1);
    else if (pieces <= 256) TALOS_POL(64, 4);
    else if (pieces <= 512) TALOS_POL(64, 8);
    else if (pieces <= 1024) TALOS_POL(256, 4);
    else if (pieces <= 2048) TALOS_POL(256, 8);
    else TALOS_POL(1024, 4);
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
