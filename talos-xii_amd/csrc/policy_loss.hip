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
// together. L lanes hold a row, V pieces each: 8 lanes up to 32 (fp32) or 64 (bf16) actions, a wave, four
// waves or sixteen beyond, up to 65536 fp32 or 131072 bf16 columns; wider rows are read again. The sums
// are fp32 (at most a few dozen terms a lane, then a tree), all that follows from them is f64.
//
// Rows of weight 0 are padding: their logits are not read, their gradient is zero.
#include <algorithm>

#include "vecio.hpp"

namespace talos {

namespace {

// partial sums of a workgroup: the loss, then the entries of enum talos_policy_stat
constexpr int kPolParts = 1 + TALOS_POLICY_NSTATS;
constexpr int kPolicyMaxVocab = 1 << 26;

struct PolicyArgs {
  int rows, vocab;
  float clip_low, clip_high, kl_coef;
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

// From the row's maximum, the sum of its exponentials and the taken logit. An action out of range has no
// log-probability: a NaN loss and no gradient.
__device__ __forceinline__ RowTerms policy_row(const PolicyArgs& a, int row, bool bad, float top, float sum,
                                               float taken) {
  RowTerms t;
  const double w = a.weight ? (double)a.weight[row] : 1.0 / (double)a.rows;
  const double logp = bad ? (double)NAN : ((double)taken - (double)top) - log((double)sum);
  const double adv = a.adv[row], diff = logp - (double)a.old_logp[row], ratio = exp(diff);
  const double lo = 1.0 - (double)a.clip_low, hi = 1.0 + (double)a.clip_high;
  // comparisons that keep a NaN ratio a NaN; ties take the clipped side
  const double plain = ratio * adv, held = (ratio < lo ? lo : ratio > hi ? hi : ratio) * adv;
  const double gain = plain < held ? plain : held;
  const bool clipped = adv >= 0.0 ? ratio > hi : ratio < lo;
  double kl = 0.0, dkl = 0.0;
  if (a.ref_logp) {
    const double gap = (double)a.ref_logp[row] - logp, e = exp(gap);
    kl = e - gap - 1.0;
    dkl = 1.0 - e;
  }
  t.sums[0] = bad ? (double)NAN : w * ((double)a.kl_coef * kl - gain);
  t.sums[1 + TALOS_POLICY_STAT_KL] = (ratio - 1.0) - diff;
  t.sums[1 + TALOS_POLICY_STAT_POLICY] = gain;
  t.sums[1 + TALOS_POLICY_STAT_REF_KL] = kl;
  t.sums[1 + TALOS_POLICY_STAT_CLIPPED] = clipped ? 1.0 : 0.0;
  t.sums[1 + TALOS_POLICY_STAT_COUNT] = 1.0;
  t.slope = bad ? 0.f : (float)(w * ((double)a.kl_coef * dkl - (clipped ? 0.0 : adv * ratio)));
  t.logp = (float)logp;
  return t;
}

// Maximum and sum over the W waves of a row's lanes (W > 1: the workgroup's own row).
template <int W>
__device__ __forceinline__ float waves_max(float v, float* red) {
  if constexpr (W == 1) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = red[0];
#pragma unroll
  for (int i = 1; i < W; ++i) t = fmaxf(t, red[i]);
  return t;
}
template <int W>
__device__ __forceinline__ float waves_sum(float v, float* red) {
  if constexpr (W == 1) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) t += red[i];
  return t;
}

// One row per L lanes. V > 0: the row stays in registers, V pieces a lane; V = 0: any width, read again
// for the gradient (L = 1024). dlogits null: the loss alone. dlogits may be the logits' own rows.
template <typename T, int L, int V>
__global__ __launch_bounds__(L > 256 ? L : 256) void policy_loss_kernel(PolicyArgs a, const T* logits, T* dlogits) {
  constexpr int N = Piece<T>::N, TB = L > 256 ? L : 256, R = TB / L, W = L > 64 ? L / 64 : 1;
  constexpr int LW = L < 64 ? L : 64;
  __shared__ float red[W];
  __shared__ double part[R][kPolParts];
  const int lane = threadIdx.x % L, sub = threadIdx.x / L;
  const long long row = (long long)blockIdx.x * R + sub;
  const bool on = row < a.rows && (!a.weight || a.weight[row] != 0.f);  // W > 1: uniform over the workgroup
  const bool in = row < a.rows;
  const T* xr = logits + (in ? row : 0) * a.ld;
  T* dr = dlogits ? dlogits + (in ? row : 0) * a.ld_d : nullptr;
  RowTerms t{};
  float top = -INFINITY, sum = 0.f;
  int act = -1;
  typename Piece<T>::Raw raw[V ? V : 1];
  if (on) {
    act = a.actions[row];
    const bool bad = act < 0 || act >= a.vocab;
    const float taken = bad ? 0.f : to_f32(xr[act]);
    // values past the row are -inf: no maximum, no share of the sum
    auto each = [&](auto&& f) {
      if constexpr (V > 0) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float v[N];
          // opaque to the compiler, which would otherwise widen the row once and hold it so (232 spills)
#pragma unroll
          for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(raw[j].w[i]));
          Piece<T>::widen(raw[j], v);
          f(v);
        }
      } else {
        for (int c = N * lane; c < a.vocab; c += N * L) {
          float v[N];
          load_piece(xr, c, a.vocab, v, -INFINITY);
          f(v);
        }
      }
    };
    if constexpr (V > 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = N * (lane + L * j);
        if (c + N <= a.vocab) {
          raw[j] = *reinterpret_cast<const typename Piece<T>::Raw*>(xr + c);
        } else {
          float v[N];
          load_piece(xr, c, a.vocab, v, -INFINITY);
          raw[j] = Piece<T>::pack(v);
        }
      }
    }
    each([&](const float(&v)[N]) {
#pragma unroll
      for (int i = 0; i < N; ++i) top = fmaxf(top, v[i]);
    });
    top = waves_max<W>(lanes_max<LW>(top), red);
    each([&](const float(&v)[N]) {
#pragma unroll
      for (int i = 0; i < N; ++i) sum += __expf(v[i] - top);
    });
    sum = waves_sum<W>(lanes_sum<LW>(sum), red);
    t = policy_row(a, (int)row, bad, top, sum, taken);
  }
  if (in && lane == 0) {
    if (a.logp) a.logp[row] = t.logp;
  }
  if (a.part) {
    if (lane == 0)
      for (int i = 0; i < kPolParts; ++i) part[sub][i] = t.sums[i];
    __syncthreads();
    if (threadIdx.x < kPolParts) {
      double s = 0.0;
      for (int r = 0; r < R; ++r) s += part[r][threadIdx.x];
      a.part[(size_t)blockIdx.x * kPolParts + threadIdx.x] = s;
    }
  }
  if (!in || !dr) return;
  const float scale = -t.slope / sum;
  auto grad = [&](float (&v)[N], int c) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = on ? __expf(v[i] - top) * scale : 0.f;
      if (on && c + i == act) v[i] += t.slope;
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
    for (int c = N * lane; c < a.vocab; c += N * L) {
      float v[N] = {};
      if (on) load_piece(xr, c, a.vocab, v);
      grad(v, c);
    }
  }
}

// The partial rows' sums in a fixed order: wave i of the workgroup takes quantity i, each lane every 64th
// partial, then the lanes' tree.
__global__ __launch_bounds__(64 * kPolParts) void policy_loss_final_kernel(int nblk, const double* __restrict__ part,
                                                                           float* __restrict__ loss, double* stats,
                                                                           int accumulate) {
  const int lane = threadIdx.x & 63, i = threadIdx.x >> 6;
  double s = 0.0;
  for (int k = lane; k < nblk; k += 64) s += part[(size_t)k * kPolParts + i];
  s = wave_sum(s);
  if (lane != 0) return;
  if (i == 0) {
    if (loss) loss[0] = (float)s;
  } else if (stats) {
    stats[i - 1] = (accumulate ? stats[i - 1] : 0.0) + s;
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
  TALOS_REQUIRE(accumulate == 0 || accumulate == 1, TALOS_ERR_SHAPE, "%s: stats_accumulate must be 0 or 1", fn);
  TALOS_REQUIRE(rows == 0 || (logits && actions && adv && old_logp), TALOS_ERR_NULL, "%s: null input", fn);
  TALOS_REQUIRE(kl_coef == 0.f || ref_logp || rows == 0, TALOS_ERR_NULL, "%s: kl_coef without ref_logp", fn);
  TALOS_DEVICE();
  constexpr int N = Piece<T>::N;
  const int pieces = (vocab + N - 1) / N;
  PolicyArgs a{rows, vocab, clip_low, clip_high, kl_coef, ld, ld_d, actions, adv, old_logp, ref_logp, weight, logp,
               nullptr};
  const int per = pieces <= 8 ? 32 : pieces <= 256 ? 4 : 1;  // rows a workgroup
  const int nblk = (int)ceil_div((size_t)rows, per);
  EntryScratch ws;
  int rc = ws.acquire(loss || stats ? (size_t)nblk * kPolParts * sizeof(double) : 0, s);
  if (rc) return rc;
  a.part = static_cast<double*>(ws.ptr);
  if (nblk > 0) {
#define TALOS_POL(L, V)                                                                                          \
  hipLaunchKernelGGL((policy_loss_kernel<T, L, V>), dim3(nblk), dim3(L > 256 ? L : 256), 0, s, a, logits, dlogits)
    if (pieces <= 8) TALOS_POL(8, 1);
    else if (pieces <= 64) TALOS_POL(64, 1);
    else if (pieces <= 256) TALOS_POL(64, 4);
    else if (pieces <= 1024) TALOS_POL(256, 4);
    else if (pieces <= 2048) TALOS_POL(256, 8);
    else if (pieces <= 4096) TALOS_POL(1024, 4);
    else if (pieces <= 8192) TALOS_POL(1024, 8);
    else if (pieces <= 16384) TALOS_POL(1024, 16);
    else TALOS_POL(1024, 0);
#undef TALOS_POL
    rc = launch_status("policy_loss_kernel");
  }
  if (!rc && (loss || stats)) {
    hipLaunchKernelGGL(policy_loss_final_kernel, dim3(1), dim3(64 * kPolParts), 0, s, nblk, a.part, loss, stats,
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
