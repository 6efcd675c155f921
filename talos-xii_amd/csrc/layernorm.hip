// layernorm.hip -- layer norm forward and backward over the last dimension, fp32 or bf16 rows.
//
// y = (x - mean) * rstd * w + b, mean and the biased variance over a row, rstd = 1 / sqrt(var + eps).
// With xh = (x - mean) * rstd and h = g * w:
//   dx = rstd * (h - mean_row(h) - xh * mean_row(h * xh)),  dw = sum_rows g * xh,  db = sum_rows g.
//
// Both passes are bound by memory: a row is read once into registers, its mean and the sum of its
// centred squares are formed there (two passes over registers, so a large mean costs no digits), and
// the result is written from the same registers. Statistics and sums are fp32 or wider; a bf16 result
// is rounded once, from its fp32 value.
//
// L lanes share a row, each holding V pieces of 16 bytes: 8, 16 or 32 lanes where a row has that few
// pieces, a wave up to 2048 values, four waves up to 8192, and beyond that a loop that reads the row
// again. The backward keeps every lane's column sums in registers over the rows that its workgroup
// walks; the lanes and waves of a workgroup add theirs in LDS, and a second kernel adds the
// workgroups' fp32 partial rows in f64, in a fixed order.
#include <algorithm>

#include "vecio.hpp"

namespace talos {

namespace {

// Sum over the L lanes of a row, all of them receiving it. L = 256: the workgroup, through red[4].
template <int L>
__device__ __forceinline__ float row_sum(float v, float* red) {
  if constexpr (L <= 64) {
    return lanes_sum<L>(v);
  } else {
    v = lanes_sum<64>(v);
    __syncthreads();  // an earlier sum's readers are done with red
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
  }
}

template <typename T, int L, int V>
__global__ __launch_bounds__(256) void layernorm_fwd_kernel(int rows, int dim, float eps, const T* __restrict__ x,
                                                            const float* __restrict__ w, const float* __restrict__ b,
                                                            T* __restrict__ y, float* __restrict__ mean_out,
                                                            float* __restrict__ rstd_out) {
  constexpr int N = Piece<T>::N;
  __shared__ float red[4];
  const long long row = (long long)blockIdx.x * (256 / L) + threadIdx.x / L;
  const int lane = threadIdx.x % L;
  if (row >= rows) return;  // L = 256: the whole workgroup
  const T* xr = x + (size_t)row * dim;
  float v[V][N];
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    load_piece(xr, N * (lane + L * j), dim, v[j]);
#pragma unroll
    for (int i = 0; i < N; ++i) s += v[j][i];
  }
  const float inv = 1.0f / (float)dim;
  const float mean = row_sum<L>(s, red) * inv;
  float q = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[j][i] -= mean;
      q += N * (lane + L * j) + i < dim ? v[j][i] * v[j][i] : 0.f;
    }
  const float rstd = 1.0f / sqrtf(row_sum<L>(q, red) * inv + eps);
  if (lane == 0) {
    if (mean_out) mean_out[row] = mean;
    if (rstd_out) rstd_out[row] = rstd;
  }
  T* yr = y + (size_t)row * dim;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = N * (lane + L * j);
    if (c >= dim) continue;
    float ww[N], bb[N];
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      float t[4];
      load_piece(w, c + k, dim, t);
#pragma unroll
      for (int i = 0; i < 4; ++i) ww[k + i] = t[i];
      if (b) {
        load_piece(b, c + k, dim, t);
#pragma unroll
        for (int i = 0; i < 4; ++i) bb[k + i] = t[i];
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[j][i] = v[j][i] * rstd * ww[i] + (b ? bb[i] : 0.f);
    store_piece(yr, c, dim, v[j]);
  }
}

// Rows of any width: a workgroup a row, the row read three times (the second and third from cache).
template <typename T>
__global__ __launch_bounds__(256) void layernorm_fwd_wide_kernel(int rows, int dim, float eps, const T* __restrict__ x,
                                                                 const float* __restrict__ w,
                                                                 const float* __restrict__ b, T* __restrict__ y,
                                                                 float* __restrict__ mean_out,
                                                                 float* __restrict__ rstd_out) {
  constexpr int N = Piece<T>::N;
  __shared__ float red[4];
  const int row = blockIdx.x;
  const T* xr = x + (size_t)row * dim;
  T* yr = y + (size_t)row * dim;
  const float inv = 1.0f / (float)dim;
  float s = 0.f, q = 0.f;
  for (int c = N * threadIdx.x; c < dim; c += N * 256) {
    float v[N];
    load_piece(xr, c, dim, v);
#pragma unroll
    for (int i = 0; i < N; ++i) s += v[i];
  }
  const float mean = row_sum<256>(s, red) * inv;
  for (int c = N * threadIdx.x; c < dim; c += N * 256) {
    float v[N];
    load_piece(xr, c, dim, v);
#pragma unroll
    for (int i = 0; i < N; ++i) q += c + i < dim ? (v[i] - mean) * (v[i] - mean) : 0.f;
  }
  const float rstd = 1.0f / sqrtf(row_sum<256>(q, red) * inv + eps);
  if (threadIdx.x == 0) {
    if (mean_out) mean_out[row] = mean;
    if (rstd_out) rstd_out[row] = rstd;
  }
  for (int c = N * threadIdx.x; c < dim; c += N * 256) {
    float v[N];
    load_piece(xr, c, dim, v);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c + i < dim) v[i] = (v[i] - mean) * rstd * w[c + i] + (b ? b[c + i] : 0.f);
    store_piece(yr, c, dim, v);
  }
}

// part: [gridDim.x][2 * dim] fp32, this workgroup's sums of g * xh, then of g (null: neither is wanted).
template <typename T, int L, int V>
__global__ __launch_bounds__(256) void layernorm_bwd_kernel(int rows, int dim, const T* __restrict__ x,
                                                            const float* __restrict__ w,
                                                            const float* __restrict__ mean,
                                                            const float* __restrict__ rstd, const T* dy,
                                                            int accumulate, T* dx, float* __restrict__ part) {
  constexpr int N = Piece<T>::N, R = 256 / L;  // rows a workgroup takes at once
  __shared__ float red[8];
  __shared__ float cols[L == 256 ? 1 : 4 * 64 * N];
  const int lane = threadIdx.x % L, sub = threadIdx.x / L;
  const float inv = 1.0f / (float)dim;
  float ww[V][N], sw[V][N], sb[V][N];
#pragma unroll
  for (int j = 0; j < V; ++j) {
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      float t[4];
      load_piece(w, N * (lane + L * j) + k, dim, t);
#pragma unroll
      for (int i = 0; i < 4; ++i) ww[j][k + i] = t[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) sw[j][i] = sb[j][i] = 0.f;
  }
  for (long long row0 = (long long)blockIdx.x * R; row0 < rows; row0 += gridDim.x * R) {
    const long long row = row0 + sub;
    const bool on = row < rows;  // L = 256: always
    float xh[V][N], g[V][N];
    const float m = on ? mean[row] : 0.f, r = on ? rstd[row] : 0.f;
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = on ? N * (lane + L * j) : dim;
      load_piece(x + (size_t)(on ? row : 0) * dim, c, dim, xh[j]);
      load_piece(dy + (size_t)(on ? row : 0) * dim, c, dim, g[j]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        xh[j][i] = (xh[j][i] - m) * r;  // g is 0 past the row, so what xh holds there does not count
        sw[j][i] += g[j][i] * xh[j][i];
        sb[j][i] += g[j][i];
        g[j][i] *= ww[j][i];
        s += g[j][i];
        q += g[j][i] * xh[j][i];
      }
    if constexpr (L <= 64) {
      s = lanes_sum<L>(s);
      q = lanes_sum<L>(q);
    } else {
      s = lanes_sum<64>(s);
      q = lanes_sum<64>(q);
      __syncthreads();
      if ((threadIdx.x & 63) == 0) {
        red[threadIdx.x >> 6] = s;
        red[4 + (threadIdx.x >> 6)] = q;
      }
      __syncthreads();
      s = (red[0] + red[1]) + (red[2] + red[3]);
      q = (red[4] + red[5]) + (red[6] + red[7]);
    }
    s *= inv;
    q *= inv;
    if (on) {
      T* dr = dx + (size_t)row * dim;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = N * (lane + L * j);
        if (c >= dim) continue;
        float o[N];
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = r * (g[j][i] - s - xh[j][i] * q);
        if (accumulate) {
          float old[N];
          load_piece(dr, c, dim, old);
#pragma unroll
          for (int i = 0; i < N; ++i) o[i] += old[i];
        }
        store_piece(dr, c, dim, o);
      }
    }
  }
  if (part == nullptr) return;
  float* p = part + (size_t)blockIdx.x * 2 * dim;
  if constexpr (L == 256) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      store_piece(p, N * (lane + L * j), dim, *reinterpret_cast<float(*)[4]>(sw[j]));
      if constexpr (N == 8) store_piece(p, N * (lane + L * j) + 4, dim, *reinterpret_cast<float(*)[4]>(sw[j] + 4));
      store_piece(p + dim, N * (lane + L * j), dim, *reinterpret_cast<float(*)[4]>(sb[j]));
      if constexpr (N == 8)
        store_piece(p + dim, N * (lane + L * j) + 4, dim, *reinterpret_cast<float(*)[4]>(sb[j] + 4));
    }
  } else {
    // the rows of a wave, then its four waves, piece by piece
    const int wv = threadIdx.x >> 6, l64 = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        float(&a)[N] = which ? sb[j] : sw[j];
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
          for (int o = L; o < 64; o <<= 1) a[i] += __shfl_xor(a[i], o, kWave);
          cols[(wv * N + i) * 64 + l64] = a[i];
        }
        __syncthreads();
        for (int e = threadIdx.x; e < L * N; e += 256) {
          const int l = e / N, i = e % N, c = N * (l + L * j) + i;
          if (c < dim)
            p[which * dim + c] = (cols[i * 64 + l] + cols[(N + i) * 64 + l]) +
                                 (cols[(2 * N + i) * 64 + l] + cols[(3 * N + i) * 64 + l]);
        }
        __syncthreads();
      }
  }
}

// dx of rows of any width: a workgroup a row, the row read twice.
template <typename T>
__global__ __launch_bounds__(256) void layernorm_bwd_wide_kernel(int rows, int dim, const T* __restrict__ x,
                                                                 const float* __restrict__ w,
                                                                 const float* __restrict__ mean,
                                                                 const float* __restrict__ rstd,
                                                                 const T* dy, int accumulate, T* dx) {
  constexpr int N = Piece<T>::N;
  __shared__ float red[4];
  const int row = blockIdx.x;
  const T *xr = x + (size_t)row * dim, *gr = dy + (size_t)row * dim;
  T* dr = dx + (size_t)row * dim;
  const float inv = 1.0f / (float)dim, m = mean[row], r = rstd[row];
  float s = 0.f, q = 0.f;
  for (int c = N * threadIdx.x; c < dim; c += N * 256) {
    float v[N], g[N];
    load_piece(xr, c, dim, v);
    load_piece(gr, c, dim, g);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float h = c + i < dim ? g[i] * w[c + i] : 0.f;
      s += h;
      q += h * ((v[i] - m) * r);
    }
  }
  s = row_sum<256>(s, red) * inv;
  q = row_sum<256>(q, red) * inv;
  for (int c = N * threadIdx.x; c < dim; c += N * 256) {
    float v[N], g[N], o[N];
    load_piece(xr, c, dim, v);
    load_piece(gr, c, dim, g);
    if (accumulate) load_piece(dr, c, dim, o);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c + i < dim) {
        const float d = r * (g[i] * w[c + i] - s - (v[i] - m) * r * q);
        o[i] = accumulate ? o[i] + d : d;
      }
    store_piece(dr, c, dim, o);
  }
}
// its column sums: workgroup (x, y) takes 64 columns over every gridDim.y-th group of four rows
template <typename T>
__global__ __launch_bounds__(256) void layernorm_cols_wide_kernel(int rows, int dim, const T* __restrict__ x,
                                                                  const float* __restrict__ mean,
                                                                  const float* __restrict__ rstd,
                                                                  const T* __restrict__ dy, float* __restrict__ part) {
  __shared__ float red[2][4][64];
  const int l = threadIdx.x & 63, wv = threadIdx.x >> 6, c = blockIdx.x * 64 + l;
  float sw = 0.f, sb = 0.f;
  if (c < dim)
    for (long long row = blockIdx.y * 4 + wv; row < rows; row += gridDim.y * 4) {
      const float g = to_f32(dy[(size_t)row * dim + c]);
      sw += g * ((to_f32(x[(size_t)row * dim + c]) - mean[row]) * rstd[row]);
      sb += g;
    }
  red[0][wv][l] = sw;
  red[1][wv][l] = sb;
  __syncthreads();
  if (wv < 2 && c < dim)
    part[(size_t)blockIdx.y * 2 * dim + (size_t)wv * dim + c] =
        (red[wv][0][l] + red[wv][1][l]) + (red[wv][2][l] + red[wv][3][l]);
}

// dw, db = beta * (dw, db) + the sum of nparts fp32 partial rows, in f64 and in a fixed order: 64 columns a
// workgroup, its 16 waves every 16th partial row.
__global__ __launch_bounds__(1024) void layernorm_parts_kernel(int dim, int nparts, const float* __restrict__ part,
                                                               float beta, float* dw, float* db) {
  __shared__ double red[16][64];
  const int l = threadIdx.x & 63, wv = threadIdx.x >> 6, c = blockIdx.x * 64 + l, n = 2 * dim;
  double s = 0.0;
  if (c < n)
    for (int p = wv; p < nparts; p += 16) s += (double)part[(size_t)p * n + c];
  red[wv][l] = s;
  __syncthreads();
  if (wv != 0 || c >= n) return;
  s = 0.0;
#pragma unroll
  for (int i = 0; i < 16; ++i) s += red[i][l];
  float* o = c < dim ? (dw ? dw + c : nullptr) : (db ? db + (c - dim) : nullptr);
  if (o) *o = (float)(s + (beta != 0.f ? (double)*o : 0.0));
}

// Workgroups of the backward: two a compute unit hold the rows in flight that memory needs, and each
// writes one partial row.
constexpr int kLnBlocks = 512;
constexpr int kLnWideParts = 64;
constexpr int kLnMaxDim = 1 << 26;

// f(L, V) with the lanes a row and the pieces a lane for `dim`; false beyond 8192 values.
template <typename T, typename F>
bool pick_shape(int dim, F&& f) {
  constexpr int N = Piece<T>::N;
  const int pieces = (dim + N - 1) / N;
#define TALOS_LN_SHAPE(L, V)                                               \
  if (pieces <= L * V) {                                                   \
    f(std::integral_constant<int, L>(), std::integral_constant<int, V>()); \
    return true;                                                           \
  }
  TALOS_LN_SHAPE(8, 1)
  TALOS_LN_SHAPE(16, 1)
  TALOS_LN_SHAPE(32, 1)
  TALOS_LN_SHAPE(64, 1)
  TALOS_LN_SHAPE(64, 2)
  TALOS_LN_SHAPE(64, 4)
  if constexpr (N == 4) {
    TALOS_LN_SHAPE(64, 8)
    TALOS_LN_SHAPE(256, 4)
    TALOS_LN_SHAPE(256, 8)
  } else {
    TALOS_LN_SHAPE(256, 2)
    TALOS_LN_SHAPE(256, 4)
  }
#undef TALOS_LN_SHAPE
  return false;
}

template <typename T>
int bwd_blocks(int rows, int dim) {
  int per = 1;
  const bool held = pick_shape<T>(dim, [&](auto L, auto) { per = 256 / decltype(L)::value; });
  if (!held) return std::min<int>(kLnWideParts, (int)ceil_div(rows, 4));
  return std::min<int>(kLnBlocks, (int)ceil_div(rows, per));
}

template <typename T>
int layernorm_fwd(const char* fn, int rows, int dim, float eps, const T* x, const float* w, const float* b, T* y,
                  float* mean, float* rstd, hipStream_t s) {
  TALOS_REQUIRE(x && w && y, TALOS_ERR_NULL, "%s: null x, w or y", fn);
  TALOS_REQUIRE(rows >= 0 && dim > 0, TALOS_ERR_SHAPE, "%s: bad shape rows=%d dim=%d", fn, rows, dim);
  TALOS_REQUIRE(eps >= 0.f, TALOS_ERR_SHAPE, "%s: eps must be >= 0", fn);
  TALOS_REQUIRE(dim <= kLnMaxDim, TALOS_ERR_UNSUPPORTED, "%s: dim %d exceeds %d", fn, dim, kLnMaxDim);
  TALOS_DEVICE();
  if (rows == 0) return entry_done(TALOS_OK, s);
  const bool held = pick_shape<T>(dim, [&](auto L, auto V) {
    constexpr int kL = decltype(L)::value, kV = decltype(V)::value;
    hipLaunchKernelGGL((layernorm_fwd_kernel<T, kL, kV>), dim3(ceil_div(rows, 256 / kL)), dim3(256), 0, s, rows, dim,
                       eps, x, w, b, y, mean, rstd);
  });
  if (!held)
    hipLaunchKernelGGL(layernorm_fwd_wide_kernel<T>, dim3(rows), dim3(256), 0, s, rows, dim, eps, x, w, b, y, mean,
                       rstd);
  return entry_done(launch_status("layernorm_fwd"), s);
}

template <typename T>
int layernorm_bwd(const char* fn, int rows, int dim, const T* x, const float* w, const float* mean, const float* rstd,
                  const T* dy, float beta_dx, T* dx, float beta_dw, float* dw, float* db, hipStream_t s) {
  TALOS_REQUIRE(x && w && mean && rstd && dy && dx, TALOS_ERR_NULL, "%s: null x, w, mean, rstd, dy or dx", fn);
  TALOS_REQUIRE(rows >= 0 && dim > 0, TALOS_ERR_SHAPE, "%s: bad shape rows=%d dim=%d", fn, rows, dim);
  TALOS_REQUIRE((beta_dx == 0.f || beta_dx == 1.f) && (beta_dw == 0.f || beta_dw == 1.f), TALOS_ERR_UNSUPPORTED,
                "%s: beta_dx / beta_dw must be 0 or 1", fn);
  TALOS_REQUIRE(dim <= kLnMaxDim, TALOS_ERR_UNSUPPORTED, "%s: dim %d exceeds %d", fn, dim, kLnMaxDim);
  TALOS_DEVICE();
  const bool sums = dw || db;
  const int nblk = rows > 0 ? bwd_blocks<T>(rows, dim) : 0;
  EntryScratch ws;
  int rc = ws.acquire(sums ? (size_t)nblk * 2 * dim * sizeof(float) : 0, s);
  if (rc) return rc;
  float* part = static_cast<float*>(ws.ptr);
  if (rows > 0) {
    const bool held = pick_shape<T>(dim, [&](auto L, auto V) {
      hipLaunchKernelGGL((layernorm_bwd_kernel<T, decltype(L)::value, decltype(V)::value>), dim3(nblk), dim3(256), 0,
                         s, rows, dim, x, w, mean, rstd, dy, beta_dx != 0.f, dx, part);
    });
    if (!held) {
      // the column sums first: dx may be dy's own buffer
      if (sums)
        hipLaunchKernelGGL(layernorm_cols_wide_kernel<T>, dim3(ceil_div(dim, 64), nblk), dim3(256), 0, s, rows, dim, x,
                           mean, rstd, dy, part);
      hipLaunchKernelGGL(layernorm_bwd_wide_kernel<T>, dim3(rows), dim3(256), 0, s, rows, dim, x, w, mean, rstd, dy,
                         beta_dx != 0.f, dx);
    }
    rc = launch_status("layernorm_bwd");
  }
  if (!rc && sums) {
    hipLaunchKernelGGL(layernorm_parts_kernel, dim3(ceil_div((size_t)2 * dim, 64)), dim3(1024), 0, s, dim, nblk, part,
                       beta_dw, dw, db);
    rc = launch_status("layernorm_parts_kernel");
  }
  const int rel = ws.release();
  return entry_done(rc ? rc : rel, s);
}

}  // namespace
}  // namespace talos

using namespace talos;

extern "C" {

int talos_layernorm_fwd_f32(int rows, int dim, float eps, const float* x, const float* w, const float* b, float* y,
                            float* mean, float* rstd, talos_stream_t stream) {
  return layernorm_fwd(__func__, rows, dim, eps, x, w, b, y, mean, rstd, as_stream(stream));
}
int talos_layernorm_fwd_bf16(int rows, int dim, float eps, const talos_bf16* x, const float* w, const float* b,
                             talos_bf16* y, float* mean, float* rstd, talos_stream_t stream) {
  return layernorm_fwd(__func__, rows, dim, eps, reinterpret_cast<const Bf16*>(x), w, b, reinterpret_cast<Bf16*>(y),
                       mean, rstd, as_stream(stream));
}
int talos_layernorm_bwd_f32(int rows, int dim, const float* x, const float* w, const float* mean, const float* rstd,
                            const float* dy, float beta_dx, float* dx, float beta_dw, float* dw, float* db,
                            talos_stream_t stream) {
  return layernorm_bwd(__func__, rows, dim, x, w, mean, rstd, dy, beta_dx, dx, beta_dw, dw, db, as_stream(stream));
}
int talos_layernorm_bwd_bf16(int rows, int dim, const talos_bf16* x, const float* w, const float* mean,
                             const float* rstd, const talos_bf16* dy, float beta_dx, talos_bf16* dx, float beta_dw,
                             float* dw, float* db, talos_stream_t stream) {
  return layernorm_bwd(__func__, rows, dim, reinterpret_cast<const Bf16*>(x), w, mean, rstd,
                       reinterpret_cast<const Bf16*>(dy), beta_dx, reinterpret_cast<Bf16*>(dx), beta_dw, dw, db,
                       as_stream(stream));
}

}  // extern "C"
