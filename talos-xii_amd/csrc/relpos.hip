// relpos.hip -- a learned relative position bias by buckets: the table of one value per (bucket, head)
// expanded to a bias by distance, which talos_gqa_* adds to the scores, and the table's gradient.
//
// A distance d = key position - query position has a bucket. Of a side's S buckets (all of them, or half
// where both directions have their own) the first E = S / 2 hold one distance each; the rest split
// E .. M = max_distance evenly by logarithm, and every distance from M on shares the last:
//   bucket(n) = n                                             n < E
//             = min(S - 1, E + floor((S - E) ln(n / E) / ln(M / E)))   n >= E
// with n = |d|, the keys after the query in the second half of the buckets, or n = max(0, -d) for one
// direction. The logarithms are f64 with 1e-9 added before the floor, so that a distance that stands
// exactly on a border (n = 2 E, 4 E, ... for the usual powers of two) belongs to the bucket that begins
// there; no other whole distance comes within 1e-9 of one for any size a caller would use.
//
// So every bucket holds one run of distances, and the bias row of a head is [2 M + 1] values: d = -M .. M.
// The gradient of a table entry is the sum of its run. Both are a few kilobytes: launch latency is all.
#include <cmath>

#include "common.hpp"

namespace talos {

namespace {

struct RelposArgs {
  int buckets, heads, max_distance, both;
  double per_log;  // (S - E) / ln(M / E)
};

__device__ __forceinline__ int relpos_bucket(const RelposArgs& a, int d) {
  const int side = a.both ? a.buckets / 2 : a.buckets, few = side / 2;
  const int n = a.both ? abs(d) : max(0, -d);
  int b = n;
  if (n >= few) {
    const double step = log((double)n / (double)few) * a.per_log + 1e-9;
    b = n >= a.max_distance ? side - 1 : min(side - 1, few + (int)step);
  }
  return b + (a.both && d > 0 ? side : 0);
}

// workgroup (x, h): 256 distances of head h
__global__ __launch_bounds__(256) void relpos_fwd_kernel(RelposArgs a, const float* __restrict__ table,
                                                         float* __restrict__ bias, int32_t* __restrict__ buckets) {
  const int n = 2 * a.max_distance + 1;
  const int i = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y;
  if (i >= n) return;
  const int b = relpos_bucket(a, i - a.max_distance);
  bias[(size_t)h * n + i] = table[(size_t)b * a.heads + h];
  if (buckets && h == 0) buckets[i] = b;
}

// workgroup h: the runs' ends into LDS, then a wave a bucket sums its run in f64 (fixed order)
constexpr int kRelposMaxBuckets = 4096, kRelposMaxDistance = 1 << 20;
__global__ __launch_bounds__(256) void relpos_bwd_kernel(RelposArgs a, const float* __restrict__ dbias, float beta,
                                                         float* dtable) {
  __shared__ int first[kRelposMaxBuckets], last[kRelposMaxBuckets], of[256];
  const int n = 2 * a.max_distance + 1, h = blockIdx.x;
  for (int b = threadIdx.x; b < a.buckets; b += 256) {
    first[b] = 0;
    last[b] = -1;  // a bucket that no distance has
  }
  __syncthreads();
  // a run begins where the bucket is not the one before; 256 distances at a time, the last one's bucket handed on
  int carried = -1;
  for (int i0 = 0; i0 < n; i0 += 256) {
    const int i = i0 + threadIdx.x;
    const int b = i < n ? relpos_bucket(a, i - a.max_distance) : -1;
    of[threadIdx.x] = b;
    __syncthreads();
    const int before = threadIdx.x ? of[threadIdx.x - 1] : carried;
    if (b != before) {
      if (b >= 0) first[b] = i;
      if (before >= 0) last[before] = i - 1;
    }
    carried = of[255];
    __syncthreads();
  }
  if (threadIdx.x == 0 && carried >= 0) last[carried] = n - 1;
  __syncthreads();
  const int lane = threadIdx.x & 63;
  for (int b = threadIdx.x >> 6; b < a.buckets; b += 4) {
    double s = 0.0;
    for (int i = first[b] + lane; i <= last[b]; i += 64) s += (double)dbias[(size_t)h * n + i];
    s = wave_sum(s);
    if (lane == 0) {
      float* o = dtable + (size_t)b * a.heads + h;
      *o = (float)(s + (beta != 0.f ? (double)*o : 0.0));
    }
  }
}

int check_relpos(const char* fn, int buckets, int heads, int max_distance, int both) {
  TALOS_REQUIRE(both == 0 || both == 1, TALOS_ERR_DTYPE, "%s: bidirectional must be 0 or 1", fn);
  TALOS_REQUIRE(heads > 0, TALOS_ERR_SHAPE, "%s: heads = %d", fn, heads);
  TALOS_REQUIRE(buckets >= (both ? 4 : 2) && (!both || buckets % 2 == 0), TALOS_ERR_SHAPE,
                "%s: %d buckets (at least 2 a direction, the same number for both)", fn, buckets);
  TALOS_REQUIRE(buckets <= kRelposMaxBuckets && heads <= 65535 && max_distance <= kRelposMaxDistance,
                TALOS_ERR_UNSUPPORTED, "%s: %d buckets, %d heads or distance %d exceed %d, 65535 or %d", fn, buckets,
                heads, max_distance, kRelposMaxBuckets, kRelposMaxDistance);
  TALOS_REQUIRE(max_distance > (both ? buckets / 4 : buckets / 2), TALOS_ERR_SHAPE,
                "%s: max_distance %d is within the buckets of one distance each", fn, max_distance);
  return TALOS_OK;
}

RelposArgs relpos_args(int buckets, int heads, int max_distance, int both) {
  const int side = both ? buckets / 2 : buckets, few = side / 2;
  return {buckets, heads, max_distance, both, (double)(side - few) / std::log((double)max_distance / (double)few)};
}

}  // namespace
}  // namespace talos

using namespace talos;

extern "C" {

int talos_relpos_bias_fwd_f32(int num_buckets, int heads, int max_distance, int bidirectional, const float* table,
                              float* bias, int32_t* buckets, talos_stream_t stream) {
  TALOS_NONNULL(table);
  TALOS_NONNULL(bias);
  int rc = check_relpos(__func__, num_buckets, heads, max_distance, bidirectional);
  if (rc) return rc;
  TALOS_DEVICE();
  const RelposArgs a = relpos_args(num_buckets, heads, max_distance, bidirectional);
  hipLaunchKernelGGL(relpos_fwd_kernel, dim3(ceil_div((size_t)2 * max_distance + 1, 256), heads), dim3(256), 0,
                     as_stream(stream), a, table, bias, buckets);
  return entry_done(launch_status("relpos_fwd_kernel"), as_stream(stream));
}

int talos_relpos_bias_bwd_f32(int num_buckets, int heads, int max_distance, int bidirectional, const float* dbias,
                              float beta, float* dtable, talos_stream_t stream) {
  TALOS_NONNULL(dbias);
  TALOS_NONNULL(dtable);
  int rc = check_relpos(__func__, num_buckets, heads, max_distance, bidirectional);
  if (rc) return rc;
  TALOS_REQUIRE(beta == 0.f || beta == 1.f, TALOS_ERR_UNSUPPORTED, "%s: beta must be 0 or 1", __func__);
  TALOS_DEVICE();
  const RelposArgs a = relpos_args(num_buckets, heads, max_distance, bidirectional);
  hipLaunchKernelGGL(relpos_bwd_kernel, dim3(heads), dim3(256), 0, as_stream(stream), a, dbias, beta, dtable);
  return entry_done(launch_status("relpos_bwd_kernel"), as_stream(stream));
}

}  // extern "C"
