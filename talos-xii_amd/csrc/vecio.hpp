// vecio.hpp -- 16-byte row access for operators that store fp32 or bf16 tensors: a piece of four
// fp32 or eight bf16 values, widened to fp32, at any element-aligned address. gfx950 loads and
// stores 16 bytes at any dword or byte address (the driver runs its memory units in unaligned
// mode), so rows of an odd width take the same wide accesses as aligned ones.
#pragma once

#include "common.hpp"

namespace talos {

typedef __bf16 bf16pair_t __attribute__((ext_vector_type(2)));
typedef float floatpair_t __attribute__((ext_vector_type(2)));

struct Bf16 {  // storage only; arithmetic is in fp32
  uint16_t bits;
};

// two values rounded to nearest even, lo in the low half
__device__ __forceinline__ uint32_t bf16_round2(float lo, float hi) {
  const floatpair_t v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16pair_t));
}
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(Bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }
__device__ __forceinline__ void from_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void from_f32(Bf16* p, float v) { p->bits = (uint16_t)bf16_round2(v, 0.f); }

template <typename T>
struct Piece;
template <>
struct Piece<float> {
  static constexpr int N = 4;
  struct __attribute__((packed, aligned(4))) Raw {
    uint32_t w[4];
  };
  static __device__ __forceinline__ void widen(const Raw& r, float (&o)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __uint_as_float(r.w[i]);
  }
  static __device__ __forceinline__ Raw pack(const float (&v)[4]) {
    Raw r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = __float_as_uint(v[i]);
    return r;
  }
};
template <>
struct Piece<Bf16> {
  static constexpr int N = 8;
  struct __attribute__((packed, aligned(2))) Raw {
    uint32_t w[4];
  };
  static __device__ __forceinline__ void widen(const Raw& r, float (&o)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[2 * i] = __uint_as_float(r.w[i] << 16);
      o[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ Raw pack(const float (&v)[8]) {
    Raw r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = bf16_round2(v[2 * i], v[2 * i + 1]);
    return r;
  }
};

// Values c .. c + N - 1 of a row of `dim` values, `fill` past its end (a piece across the end goes
// value by value, so nothing past the row is read or written).
template <typename T>
__device__ __forceinline__ void load_piece(const T* row, int c, int dim, float (&o)[Piece<T>::N], float fill = 0.f) {
  constexpr int N = Piece<T>::N;
  if (c + N <= dim) {
    Piece<T>::widen(*reinterpret_cast<const typename Piece<T>::Raw*>(row + c), o);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = c + i < dim ? to_f32(row[c + i]) : fill;
  }
}
// The piece as it is in memory, `fill` (a value of T that survives the round trip) past the row's end.
template <typename T>
__device__ __forceinline__ typename Piece<T>::Raw load_raw(const T* row, int c, int dim, float fill = 0.f) {
  if (c + Piece<T>::N <= dim) return *reinterpret_cast<const typename Piece<T>::Raw*>(row + c);
  float v[Piece<T>::N];
  load_piece(row, c, dim, v, fill);
  return Piece<T>::pack(v);
}
// The same in two steps, so that the loads of many pieces are in flight together and none is waited for where it is issued
// (a piece across the end, loaded value by value, is): row_piece loads the piece, or the row's last N values where it would
// pass its end; row_piece_end moves those into place, `fill` behind them. (13421 rows of 2500 bf16 values, layer norm
// forward and backward: 40 + 87 us with load_raw, 30 + 50 so; 7666 of 4377: 42 + 83, 33 + 58.)
template <typename T>
__device__ __forceinline__ typename Piece<T>::Raw row_piece(const T* row, int c, int dim, float fill = 0.f) {
  if (dim < Piece<T>::N) return load_raw(row, c, dim, fill);
  return *reinterpret_cast<const typename Piece<T>::Raw*>(row + min(c, dim - Piece<T>::N));
}
template <typename T>
__device__ __forceinline__ void row_piece_end(typename Piece<T>::Raw& r, int c, int dim, float fill = 0.f) {
  constexpr int N = Piece<T>::N, P = N / 4;  // values a piece, a word
  const int over = c + N - dim;              // values past the end
  if (over <= 0) return;
  const uint32_t none = P == 1 ? __float_as_uint(fill) : bf16_round2(fill, fill);
  auto words = [&](int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = i + n < 4 ? r.w[(i + n) & 3] : none;
  };
  if (over >= N) {
    words(4);
    return;
  }
  if (dim < N) return;
  if (over & (2 * P)) words(2);
  if (over & P) words(1);
  if (P == 2 && (over & 1)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = r.w[i] >> 16 | (i < 3 ? r.w[(i + 1) & 3] : none) << 16;
  }
}
template <typename T>
__device__ __forceinline__ void store_piece(T* row, int c, int dim, const float (&v)[Piece<T>::N]) {
  constexpr int N = Piece<T>::N;
  if (c + N <= dim) {
    *reinterpret_cast<typename Piece<T>::Raw*>(row + c) = Piece<T>::pack(v);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c + i < dim) from_f32(row + c + i, v[i]);
  }
}

// Sum (or maximum) over the L lanes that share a row, L a power of two up to 64.
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}
template <int L>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, kWave));
  return v;
}

}  // namespace talos
