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
// pieces, a wave up to 1024 values, more waves up to 8192 (pick_shape), and beyond that a loop that reads
// the row again. The backward keeps every lane's column sums in registers over the rows that its workgroup
// walks; the lanes and waves of a workgroup add theirs in LDS, and a second kernel adds the
// workgroups' fp32 partial rows in f64, in a fixed order.
#include <algorithm>

#include "vecio.hpp"

namespace talos {

namespace {

// Threads of a workgroup whose rows take L lanes.
template <int L>
constexpr int kLnThreads = L > 256 ? L : 256;

// Sums of a and b over the L lanes of a row, all of them receiving them. L > 64: the workgroup, through red[2 L / 64].
template <int L>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* red) {
  if constexpr (L <= 64) {
    a = lanes_sum<L>(a);
    b = lanes_sum<L>(b);
  } else {
    constexpr int W = L / 64;
    a = lanes_sum<64>(a);
    b = lanes_sum<64>(b);
    __syncthreads();  // an earlier sum's readers are done with red
    if ((threadIdx.x & 63) == 0) {
      red[threadIdx.x >> 6] = a;
      red[W + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      a += red[i];
      b += red[W + i];
    }
  }
}
template <int L>
__device__ __forceinline__ float row_sum(float v, float* red) {
  float none = 0.f;
  row_sum2<L>(v, none, red);
  return v;
}

// w and b stay in registers over the rows that a workgroup walks (read with every row they are four times a bf16 row's own
// bytes: 8192 x 4096 bf16 37.4 us, 23.7 held), and the next row is on its way while one is reduced and written.
template <typename T, int L, int V>
__global__ __launch_bounds__(kLnThreads<L>) void layernorm_fwd_kernel(int rows, int dim, float eps, const T* x,
                                                                      const float* __restrict__ w,
                                                                      const float* __restrict__ b, T* y,
                                                                      float* __restrict__ mean_out,
                                                                      float* __restrict__ rstd_out) {
  constexpr int N = Piece<T>::N, R = kLnThreads<L> / L;
  __shared__ float red[L > 64 ? 2 * L / 64 : 1];
  const int lane = threadIdx.x % L, sub = threadIdx.x / L;
  const float inv = 1.0f / (float)dim;
  float ww[V][N], bb[V][N];
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int p = 0; p < N; p += 4) {
      float t[4] = {};
      load_piece(w, N * (lane + L * j) + p, dim, t);
#pragma unroll
      for (int i = 0; i < 4; ++i) ww[j][p + i] = t[i];
      if (b) load_piece(b, N * (lane + L * j) + p, dim, t);
#pragma unroll
      for (int i = 0; i < 4; ++i) bb[j][p + i] = b ? t[i] : 0.f;
    }
  typename Piece<T>::Raw next[V];
  auto fetch = [&](long long row) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      next[j] = row_piece(x + (size_t)(row < rows ? row : 0) * dim, N * (lane + L * j), dim);
  };
  const long long step = (long long)gridDim.x * R;
  fetch((long long)blockIdx.x * R + sub);
  for (long long row0 = (long long)blockIdx.x * R; row0 < rows; row0 += step) {
    const long long row = row0 + sub;
    float v[V][N];
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      row_piece_end<T>(next[j], N * (lane + L * j), dim);
      Piece<T>::widen(next[j], v[j]);
#pragma unroll
      for (int i = 0; i < N; ++i) s += v[j][i];
    }
    if (row0 + step < rows) fetch(row + step);
    const float mean = row_sum<L>(s, red) * inv;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[j][i] -= mean;
        q += N * (lane + L * j) + i < dim ? v[j][i] * v[j][i] : 0.f;
      }
    const float rstd = 1.0f / sqrtf(row_sum<L>(q, red) * inv + eps);
    if (row >= rows) continue;  // L > 64: never
    if (lane == 0) {
      if (mean_out) mean_out[row] = mean;
      if (rstd_out) rstd_out[row] = rstd;
    }
    T* yr = y + (size_t)row * dim;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = N * (lane + L * j);
      if (c >= dim) continue;
#pragma unroll
      for (int i = 0; i < N; ++i) v[j][i] = v[j][i] * rstd * ww[j][i] + bb[j][i];
      store_piece(yr, c, dim, v[j]);
    }
  }
}

// Rows of any width: a workgroup a row, the row read three times (the second and third from cache). A lane's own sums,
// up to 2^18 terms, are f64.
template <typename T>
__global__ __launch_bounds__(256) void layernorm_fwd_wide_kernel(int rows, int dim, float eps, const T* x,
                                                                 const float* __restrict__ w,
                                                                 const float* __restrict__ b, T* y,
                                                                 float* __restrict__ mean_out,
                                                                 float* __restrict__ rstd_out) {
  constexpr int N = Piece<T>::N;
  __shared__ float red[8];
  const int row = blockIdx.x;
  const T* xr = x + (size_t)row * dim;
  T* yr = y + (size_t)row * dim;
  const float inv = 1.0f / (float)dim;
  double s = 0.0, q = 0.0;
  for (int c = N * threadIdx.x; c < dim; c += N * 256) {
    float v[N];
    load_piece(xr, c, dim, v);
#pragma unroll
    for (int i = 0; i < N; ++i) s += (double)v[i];
  }
  const float mean = row_sum<256>((float)s, red) * inv;
  for (int c = N * threadIdx.x; c < dim; c += N * 256) {
    float v[N];
    load_piece(xr, c, dim, v);
#pragma unroll
    for (int i = 0; i < N; ++i) q += (double)(c + i < dim ? (v[i] - mean) * (v[i] - mean) : 0.f);
  }
  const float rstd = 1.0f / sqrtf(row_sum<256>((float)q, red) * inv + eps);
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
__global__ __launch_bounds__(kLnThreads<L>) void layernorm_bwd_kernel(int rows, int dim, const T* __restrict__ x,
                                                            const float* __restrict__ w,
                                                            const float* __restrict__ mean,
                                                            const float* __restrict__ rstd, const T* dy,
                                                            int accumulate, T* dx, float* __restrict__ part) {
  constexpr int N = Piece<T>::N, R = kLnThreads<L> / L;  // rows a workgroup takes at once
  __shared__ float red[L > 64 ? 2 * L / 64 : 1];
  __shared__ float cols[L > 64 ? 1 : 4 * 64 * N];
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
  // the next rows' pieces and statistics are on their way while a row is reduced and written
  typename Piece<T>::Raw nx[V], ng[V];
  float nm = 0.f, nr = 0.f;
  auto fetch = [&](long long row) {
    const bool on = row < rows;
    nm = on ? mean[row] : 0.f;
    nr = on ? rstd[row] : 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = N * (lane + L * j);
      nx[j] = row_piece(x + (size_t)(on ? row : 0) * dim, c, dim);
      ng[j] = row_piece(dy + (size_t)(on ? row : 0) * dim, c, dim);
    }
  };
  const long long step = (long long)gridDim.x * R;
  fetch((long long)blockIdx.x * R + sub);
  for (long long row0 = (long long)blockIdx.x * R; row0 < rows; row0 += step) {
    const long long row = row0 + sub;
    const bool on = row < rows;  // L > 64: always
    float xh[V][N], g[V][N];
    const float m = nm, r = nr;
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = on ? N * (lane + L * j) : dim;  // a row past the last: zeros
      row_piece_end<T>(nx[j], c, dim);
      row_piece_end<T>(ng[j], c, dim);
      Piece<T>::widen(nx[j], xh[j]);
      Piece<T>::widen(ng[j], g[j]);
    }
    if (row0 + step < rows) fetch(row + step);
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
    row_sum2<L>(s, q, red);
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
  if constexpr (L > 64) {
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

// dx of rows of any width: a workgroup a row, the row read twice; a lane's own sums f64.
template <typename T>
__global__ __launch_bounds__(256) void layernorm_bwd_wide_kernel(int rows, int dim, const T* __restrict__ x,
                                                                 const float* __restrict__ w,
                                                                 const float* __restrict__ mean,
                                                                 const float* __restrict__ rstd,
                                                                 const T* dy, int accumulate, T* dx) {
  constexpr int N = Piece<T>::N;
  __shared__ float red[8];
  const int row = blockIdx.x;
  const T *xr = x + (size_t)row * dim, *gr = dy + (size_t)row * dim;
  T* dr = dx + (size_t)row * dim;
  const float inv = 1.0f / (float)dim, m = mean[row], r = rstd[row];
  double s64 = 0.0, q64 = 0.0;
  for (int c = N * threadIdx.x; c < dim; c += N * 256) {
    float v[N], g[N];
    load_piece(xr, c, dim, v);
    load_piece(gr, c, dim, g);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float h = c + i < dim ? g[i] * w[c + i] : 0.f;
      s64 += (double)h;
      q64 += (double)(h * ((v[i] - m) * r));
    }
  }
  float s = (float)s64, q = (float)q64;
  row_sum2<256>(s, q, red);
  s *= inv;
  q *= inv;
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

// dw, db = beta * (dw, db) + the sum of nparts fp32 partial rows, in f64 and in a fixed order: C columns a workgroup, its
// 1024 / C groups of C lanes every 1024 / C-th partial row. C = 16 where 64 would leave most compute units idle (256
// columns of 512 partial rows: 11.0 us with 64, 4.7 with 16).
template <int C>
__global__ __launch_bounds__(1024) void layernorm_parts_kernel(int dim, int nparts, const float* __restrict__ part,
                                                               float beta, float* dw, float* db) {
  constexpr int G = 1024 / C;
  __shared__ double red[G][C + 1];
  const int l = threadIdx.x % C, g = threadIdx.x / C, c = blockIdx.x * C + l, n = 2 * dim;
  double s = 0.0;
  if (c < n)
    for (int p = g; p < nparts; p += G) s += (double)part[(size_t)p * n + c];
  red[g][l] = s;
  __syncthreads();
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    if (g < o) red[g][l] += red[g + o][l];
    __syncthreads();
  }
  if (g != 0 || c >= n) return;
  s = red[0][l];
  float* o = c < dim ? (dw ? dw + c : nullptr) : (db ? db + (c - dim) : nullptr);
  if (o) *o = (float)(s + (beta != 0.f ? (double)*o : 0.0));
}

// Workgroups of the backward, each of which writes one partial row: two a compute unit (8192 x 4096 bf16, forward and
// backward, 69 us; one 87, four 84), one where a row takes more than eight waves, of which no second set fits beside it
// (4096 x 8192 bf16, backward: 42 us; 53 with two in turn).
constexpr int kLnBlocks = 512;
constexpr int kLnWideParts = 64;
constexpr int kLnMaxDim = 1 << 26;

// f(L, V) with the lanes a row and the pieces a lane for `dim`; false beyond 8192 values. 16 values a lane at most, which
// the backward holds beside another row's and two sums a column; past 4096 values it takes 8 a lane for bf16 and fp32 alike
// (4377 bf16: 58 us, 88 with 16 in half as many lanes), the forward 16 (33 us, 42 with 8). A row of 257 to 384 pieces
// leaves fewer lanes idle in six waves: backward of 2500 bf16 50 us, 55 with four waves of twice the pieces (the
// forward 49, 30 with four).
template <typename T, bool BWD, typename F>
bool pick_shape(int dim, F&& f) {
  constexpr int N = Piece<T>::N, U = N == 4 ? 2 : 1;
  const int pieces = (dim + N - 1) / N;
#define TALOS_LN_SHAPE(L, V)                                               \
  if (pieces <= L * (V)) {                                                 \
    f(std::integral_constant<int, L>(), std::integral_constant<int, V>()); \
    return true;                                                           \
  }
  TALOS_LN_SHAPE(8, 1)
  TALOS_LN_SHAPE(16, 1)
  TALOS_LN_SHAPE(32, 1)
  TALOS_LN_SHAPE(64, 1)
  TALOS_LN_SHAPE(64, 2)
  if constexpr (N == 4) TALOS_LN_SHAPE(64, 4)
  TALOS_LN_SHAPE(256, U)
  if constexpr (BWD) TALOS_LN_SHAPE(384, U)
  TALOS_LN_SHAPE(256, 2 * U)
  if constexpr (BWD) {
    TALOS_LN_SHAPE(768, U)
    TALOS_LN_SHAPE(1024, U)
  } else {
    TALOS_LN_SHAPE(512, 2 * U)
  }
#undef TALOS_LN_SHAPE
  return false;
}

template <typename T>
int bwd_blocks(int rows, int dim) {
  int per = 1, most = kLnBlocks;
  const bool held = pick_shape<T, true>(dim, [&](auto L, auto) {
    constexpr int kL = decltype(L)::value;
    per = kLnThreads<kL> / kL;
    if (kL > 512) most = kLnBlocks / 2;
  });
  if (!held) return std::min<int>(kLnWideParts, (int)ceil_div(rows, 4));
  return std::min<int>(most, (int)ceil_div(rows, per));
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
  const bool held = pick_shape<T, false>(dim, [&](auto L, auto V) {
    constexpr int kL = decltype(L)::value, kV = decltype(V)::value;
    // 1024 threads a compute unit, half of what it holds: the rest of its registers are the rows on their way
    constexpr int kThreads = kLnThreads<kL>;
    const unsigned blocks = std::min<unsigned>(ceil_div(rows, kThreads / kL), 128 * 2048 / kThreads);
    hipLaunchKernelGGL((layernorm_fwd_kernel<T, kL, kV>), dim3(blocks), dim3(kThreads), 0, s, rows, dim, eps, x, w, b, y,
                       mean, rstd);
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
    const bool held = pick_shape<T, true>(dim, [&](auto L, auto V) {
      constexpr int kL = decltype(L)::value;
      hipLaunchKernelGGL((layernorm_bwd_kernel<T, kL, decltype(V)::value>), dim3(nblk), dim3(kLnThreads<kL>), 0, s,
                         rows, dim, x, w, mean, rstd, dy, beta_dx != 0.f, dx, part);
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
    if (dim <= 4096)
      hipLaunchKernelGGL(layernorm_parts_kernel<16>, dim3(ceil_div((size_t)2 * dim, 16)), dim3(1024), 0, s, dim, nblk, part,
                         beta_dw, dw, db);
    else
      hipLaunchKernelGGL(layernorm_parts_kernel<64>, dim3(ceil_div((size_t)2 * dim, 64)), dim3(1024), 0, s, dim, nblk, part,
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
