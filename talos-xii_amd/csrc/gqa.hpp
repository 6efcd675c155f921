// gqa.hpp -- what the grouped-query attention kernels (gqa_fwd.hip, gqa_bwd.hip) share: the arguments, the
// operands' fragments, the LDS tiles and the order in which workgroups take their tiles.
//
// Every contraction runs on v_mfma_f32_32x32x16_bf16. A bf16 tensor is its own operand. An fp32 value is
// split into three bf16 pieces (each the nearest bf16 to what the earlier ones left: exact), and a product
// is formed from the six pairs of pieces with index sum <= 2; the pairs left out are below 2^-24 of a term
// together. So both types run the same kernels, with NP = 1 or 3 planes an operand.
//
// Accumulators. Block products are laid out so that the softmaxed index runs over an accumulator's
// registers and the row that a statistic belongs to over its lanes (S^T = K Q^T, forward and dQ; S = Q K^T
// with keys over lanes for dK and dV): maxima, sums and the row's lse are then one value a lane, and the
// probabilities go straight from the accumulator into the next product's B operand. That product sums over
// rows 16 t + 8 (j / 4) + 4 h + j % 4 in slot 8 h + j (lane half h), and its A operand, the transposed
// tile, is read in that order from the row-major tile by two transposing LDS reads.
#pragma once

#include "vecio.hpp"

namespace talos {

typedef __bf16 gq_bf16x8 __attribute__((ext_vector_type(8)));
typedef float gq_f32x16 __attribute__((ext_vector_type(16)));
typedef short gq_s16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct GqaArgs {
  int B, Sq, Sk, H, KV, G, dk, dv, causal, M;
  float scale, c;  // c = scale log2(e): scores in units of log 2
  const int32_t *qlens, *klens;
  const float* bias;  // [H][2 M + 1]
  const void *q, *k, *v, *o, *dout;
  long long ldq, ldk, ldv, ldo, lddo;
  void *out, *dq, *dkey, *dval;  // the forward's o; the gradients
  long long lddq, lddk, lddv;
  float *lse, *delta;
  int tiles, splits;      // row tiles (or key tiles) a pair of sample and key head; parts a tile's loop is cut into
  float *part0, *part1;   // the parts' results where splits > 1: o or dq or dk, then lse or dv
  int few;                // keys up to which a workgroup's dQ is corrected (bf16)
  int heads_per_split;    // dK / dV: splits = (G / heads_per_split) * splits_q
  int splits_q;
  float* dbias_part;      // [B][H][tiles][splits_q][2 M + 1]
};

// the wave's number, known to the compiler to be one for all its lanes
__device__ __forceinline__ int gq_wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

template <typename T>
constexpr int kPlanes = sizeof(T) == 4 ? 3 : 1;

// Row r, 16-byte chunk c of a row-major tile of D bf16 values a row, as an element offset. The chunks of a
// row are permuted so that both kinds of read fall on distinct banks: 16 rows of one chunk (the row
// operands) and 4 rows of 4 adjacent chunks (the transposing reads). 128 wide: a row is all 64 banks, so the
// low two bits of r choose the group of four chunks and the next two the place in it; 64 wide, two rows
// share the banks, 32 wide four.
template <int D>
__device__ __forceinline__ int gq_at(int r, int c) {
  const int f = D == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : D == 64 ? ((r >> 1) & 1) << 2 | ((r >> 2) & 3) : (r >> 2) & 3;
  return r * D + ((c ^ f) << 3);
}

// Eight values of a row on their way from memory to an operand.
template <typename T>
struct Eight;
template <>
struct Eight<Bf16> {
  uint4 u;
  __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
  // values c .. c + 7 of a row of n, zero past its end
  __device__ __forceinline__ void load(const Bf16* row, int c, int n) {
    if (c + 8 <= n) {
      const Piece<Bf16>::Raw r = *reinterpret_cast<const Piece<Bf16>::Raw*>(row + c);
      u = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = c + 2 * i < n ? row[c + 2 * i].bits : 0, hi = c + 2 * i + 1 < n ? row[c + 2 * i + 1].bits : 0;
        w[i] = lo | hi << 16;
      }
      u = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __device__ __forceinline__ void planes(uint4 (&p)[1]) const { p[0] = u; }
  __device__ __forceinline__ float dot(const Eight& b) const {
    const uint32_t x[4] = {u.x, u.y, u.z, u.w}, y[4] = {b.u.x, b.u.y, b.u.z, b.u.w};
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s = fmaf(__uint_as_float(x[i] << 16), __uint_as_float(y[i] << 16), s);
      s = fmaf(__uint_as_float(x[i] & 0xffff0000u), __uint_as_float(y[i] & 0xffff0000u), s);
    }
    return s;
  }
};
// eight fp32 values to their three bf16 pieces
__device__ __forceinline__ void gq_split(const float* f, uint4 (&p)[3]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = f[i];
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = bf16_round2(r[2 * i], r[2 * i + 1]);
      if (q < 2) {
        r[2 * i] -= __uint_as_float(w[i] << 16);
        r[2 * i + 1] -= __uint_as_float(w[i] & 0xffff0000u);
      }
    }
    p[q] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
template <>
struct Eight<float> {
  float f[8];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.f;
  }
  __device__ __forceinline__ void load(const float* row, int c, int n) {
    if (c + 8 <= n) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float t[4];
        Piece<float>::widen(*reinterpret_cast<const Piece<float>::Raw*>(row + c + 4 * j), t);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[4 * j + i] = t[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = c + i < n ? row[c + i] : 0.f;
    }
  }
  __device__ __forceinline__ void planes(uint4 (&p)[3]) const { gq_split(f, p); }
  __device__ __forceinline__ float dot(const Eight& b) const {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(f[i], b.f[i], s);
    return s;
  }
};

// An operand's fragment: one 8-value piece a plane.
template <int NP>
struct Frag {
  gq_bf16x8 p[NP];
};
template <typename T>
__device__ __forceinline__ Frag<kPlanes<T>> gq_frag(const Eight<T>& e) {
  uint4 p[kPlanes<T>];
  e.planes(p);
  Frag<kPlanes<T>> f;
#pragma unroll
  for (int i = 0; i < kPlanes<T>; ++i) f.p[i] = __builtin_bit_cast(gq_bf16x8, p[i]);
  return f;
}
// eight accumulator values (probabilities or their gradients) as an operand: rounded to bf16 (NP = 1) or split
template <int NP>
__device__ __forceinline__ Frag<NP> gq_frag_acc(const float* f) {
  Frag<NP> r;
  if constexpr (NP == 1) {
    const uint4 u = {bf16_round2(f[0], f[1]), bf16_round2(f[2], f[3]), bf16_round2(f[4], f[5]), bf16_round2(f[6], f[7])};
    r.p[0] = __builtin_bit_cast(gq_bf16x8, u);
  } else {
    uint4 p[3];
    gq_split(f, p);
#pragma unroll
    for (int i = 0; i < 3; ++i) r.p[i] = __builtin_bit_cast(gq_bf16x8, p[i]);
  }
  return r;
}
// A lane's places in a tile, in bytes from its start. Row operands read row l32 (of a block of 32) and chunk 2 s + h;
// transposing reads read 4 x 16 blocks by groups of 16 lanes: lane 4 a + j of group g reads row 4 (g / 2) + a (and 8
// further) from column 16 (g % 2) + 4 j on, and receives one column of the four rows. Steps along the columns flip
// address bits above the lane's own (the chunks are permuted by XOR), steps along the rows are constants.
template <int D>
struct GqaLane {
  uint32_t row, tr;
  __device__ __forceinline__ GqaLane() {
    const int lane = threadIdx.x & 63, g = lane >> 4, a = (lane >> 2) & 3, j = lane & 3;
    row = 2 * gq_at<D>(lane & 31, lane >> 5);
    tr = 2 * (gq_at<D>(4 * (g >> 1) + a, 2 * (g & 1) + (j >> 1)) + 4 * (j & 1));
  }
  // makes the compiler form the addresses anew (an instruction each) where it would keep dozens in registers
  __device__ __forceinline__ void renew() { asm volatile("" : "+v"(row), "+v"(tr)); }
};
// chunk 2 s + h of row rb + l32 (rb a multiple of 32) of a tile whose planes are PL elements apart
template <int NP, int D, int PL>
__device__ __forceinline__ Frag<NP> gq_frag_row(const uint16_t* tile, const GqaLane<D>& ln, int rb, int s) {
  const char* at = reinterpret_cast<const char*>(tile) + (ln.row ^ (uint32_t)(32 * s)) + 2 * rb * D;
  Frag<NP> f;
#pragma unroll
  for (int i = 0; i < NP; ++i)
    f.p[i] = __builtin_bit_cast(gq_bf16x8, *reinterpret_cast<const uint4*>(at + 2 * i * PL));
  return f;
}
// The transposed tile's fragment for column block 32 ob and rows r0 + 4 h + 0..3 and r0 + 8 + 4 h + 0..3 (r0 a multiple
// of 16): lane (l32, h) gets them of column 32 ob + l32. Rows 8 further have the permutation's bit 1 flipped.
template <int NP, int D, int PL>
__device__ __forceinline__ Frag<NP> gq_frag_tr(const uint16_t* tile, const GqaLane<D>& ln, int r0, int ob) {
  typedef __attribute__((address_space(3))) gq_s16x4* lds4;
  const char* lo = reinterpret_cast<const char*>(tile) + (ln.tr ^ (uint32_t)(64 * ob)) + 2 * r0 * D;
  const char* hi = reinterpret_cast<const char*>(tile) + (ln.tr ^ (uint32_t)(64 * ob + 32)) + 2 * (r0 + 8) * D;
  Frag<NP> f;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(lo + 2 * i * PL)));
    const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(hi + 2 * i * PL)));
    f.p[i] = __builtin_bit_cast(gq_bf16x8, make_uint4(x.x, x.y, y.x, y.y));
  }
  return f;
}

__device__ __forceinline__ gq_f32x16 gq_mfma(gq_bf16x8 a, gq_bf16x8 b, gq_f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ gq_f32x16 gq_zero() {
  gq_f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}
// the five small pairs of a split product, and the leading one
__device__ __forceinline__ gq_f32x16 gq_mfma_small(const Frag<3>& a, const Frag<3>& b, gq_f32x16 c) {
  c = gq_mfma(a.p[0], b.p[2], c);
  c = gq_mfma(a.p[2], b.p[0], c);
  c = gq_mfma(a.p[1], b.p[1], c);
  c = gq_mfma(a.p[0], b.p[1], c);
  return gq_mfma(a.p[1], b.p[0], c);
}

// An accumulator whose every column holds v of its row, for lane l32's v of row l32: one product of v's three bf16
// pieces with ones. (A row's value in each of 16 registers would be four 16-byte LDS reads a lane.)
__device__ __forceinline__ gq_f32x16 gq_rows(float v, int h) {
  const uint32_t a = bf16_round2(v, 0.f) & 0xffffu;
  v -= __uint_as_float(a << 16);
  const uint32_t b = bf16_round2(v, 0.f) & 0xffffu;
  v -= __uint_as_float(b << 16);
  const uint32_t c = bf16_round2(v, 0.f) & 0xffffu;
  const uint4 x = h ? make_uint4(0, 0, 0, 0) : make_uint4(a | b << 16, c, 0, 0);
  const uint4 one = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
  return gq_mfma(__builtin_bit_cast(gq_bf16x8, x), __builtin_bit_cast(gq_bf16x8, one), gq_zero());
}

// Accumulator row of register r in lane half h (the column is lane % 32).
__device__ __forceinline__ constexpr int gq_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// The other half's value, combined: lanes l and l ^ 32.
__device__ __forceinline__ float gq_max_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float gq_sum_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A bias entry in units of log 2. The product overflows below -3.4e30, so such an entry (the type's lowest value, as masks
// are often written) hides its keys as -infinity does: where a row's every key had one, no digits of lse would be left to
// form its probabilities from again.
__device__ __forceinline__ float gq_bias(float b) { return b * 1e8f * (kLog2e * 1e-8f); }

// A sample's lengths and where its queries stand among its keys.
struct GqaSample {
  int ql, kl, off;
};
__device__ __forceinline__ GqaSample gq_sample(const GqaArgs& a, int b) {
  GqaSample s;
  s.ql = a.qlens ? __builtin_amdgcn_readfirstlane(min(max(a.qlens[b], 0), a.Sq)) : a.Sq;
  s.kl = a.klens ? __builtin_amdgcn_readfirstlane(min(max(a.klens[b], 0), a.Sk)) : a.Sk;
  s.off = s.kl - s.ql;
  return s;
}

// Which (sample, key head), tile and part a workgroup takes. Workgroups go round robin over the eight XCDs,
// each with an L2 of its own: where the pairs divide evenly among them, a pair's tiles all go to one XCD, so
// that its keys and values are read into one L2. Tiles run from the last (rev: a causal query tile's longest)
// over all pairs of an XCD before the next. Pairs count samples fastest, so samples of different lengths meet
// on an XCD.
struct GqaItem {
  int b, kvh, tile, split;
};
__device__ __forceinline__ GqaItem gq_item(const GqaArgs& a, bool rev) {
  const int pairs = a.B * a.KV;
  int id = blockIdx.x;
  GqaItem it;
  int pair, tile;
  it.split = id % a.splits;
  id /= a.splits;
  if (pairs % 8 == 0 && a.splits == 1) {
    const int mine = pairs / 8, l = id / 8;
    pair = id % 8 + 8 * (l % mine);
    tile = l / mine;
  } else {
    pair = id % pairs;
    tile = id / pairs;
  }
  it.tile = rev ? a.tiles - 1 - tile : tile;
  it.b = pair % a.B;
  it.kvh = pair / a.B;
  return it;
}

// A tile of NR rows (0 <= row0 + r < rows read, others zero) on its way to LDS: D / 8 chunks a row, PER a thread.
template <typename T, int D, int NR>
struct GqaTile {
  static constexpr int CH = D / 8, SLOTS = NR * CH, PER = (SLOTS + 255) / 256, NP = kPlanes<T>, PL = NR * D;
  Eight<T> e[PER];
  __device__ __forceinline__ void fetch(const T* base, long long ld, int row0, int rows, int n) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int s = i * 256 + (int)threadIdx.x, r = row0 + s / CH, c = 8 * (s % CH);
      if ((SLOTS % 256 == 0 || s < SLOTS) && r < rows && c < n)
        e[i].load(base + r * ld, c, n);
      else
        e[i].zero();
    }
  }
  __device__ __forceinline__ void stash(uint16_t* tile) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int s = i * 256 + (int)threadIdx.x;
      if (SLOTS % 256 != 0 && s >= SLOTS) continue;
      uint4 p[NP];
      e[i].planes(p);
#pragma unroll
      for (int q = 0; q < NP; ++q) *reinterpret_cast<uint4*>(tile + q * PL + gq_at<D>(s / CH, s % CH)) = p[q];
    }
  }
};

// The same for a bf16 tile whose rows are D values wide and 16-byte aligned, straight from memory into LDS
// (global_load_lds_dwordx4: lane i's 16 bytes go to the wave's LDS address + 16 i). No registers hold the tile and no
// LDS stores are issued. An instruction fills 64 chunks of LDS, 512 / D rows, so the permutation of chunks is made on
// the memory side: each lane fetches the chunk that belongs at its place, the same one for every instruction (the rows
// of a lane differ by multiples of 16). Rows from `rows` on are filled with the last valid one: scores against it are
// masked and probabilities of it are zero, as they are for the zero rows above.
// Issued from inline assembly, so that the compiler does not wait for all of them before every LDS read that follows;
// gq_dma_wait() and a barrier publish them. Other waits of the compiler's only get stronger by them.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void gq_dma16(const void* base, uint32_t offset, const void* lds) {
  const uint32_t to =
      __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)lds);
  const uint64_t at = (uint64_t)base;
  const uint64_t from = (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(at >> 32)) << 32 |
                        (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)at);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(from)
               : "memory", "m0");
}
#pragma clang diagnostic pop
// waits until at most N of the wave's memory instructions are in flight (those issued last)
template <int N = 0>
__device__ __forceinline__ void gq_dma_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// the wave's LDS reads have arrived: what they read may be overwritten
__device__ __forceinline__ void gq_reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// W = 4: the workgroup's waves fetch a tile together. W = 1: a wave fetches a tile of its own (the rows of a lane are then
// fewer than 16 apart, and the chunk it fetches changes with the instruction).
template <int D, int NR, int W = 4>
struct GqaDma {
  static constexpr int CH = D / 8, RPI = 64 / CH, PER = NR * CH / (64 * W);  // rows an instruction, instructions a wave
  static_assert(NR * CH % (64 * W) == 0 && (W == 1 || W * RPI % 16 == 0), "whole instructions, rows 16 apart");
  int row;                 // this lane's row of the first instruction
  uint32_t offset, chunk;  // in bytes, from the tile's first row: that row's, and the chunk's in it
  __device__ __forceinline__ void init(long long ld) {
    const int lane = threadIdx.x & 63;
    row = (W == 1 ? 0 : gq_wave() * RPI) + lane / CH;
    const int place = gq_at<D>(row, 0) / 8 % CH;  // where chunk 0 of the row stands: the row's permutation
    offset = (uint32_t)(row * ld) * 2;
    chunk = 16 * ((lane % CH) ^ place);
  }
  // rows row0 .. row0 + NR - 1 of base (row stride ld), of which `rows` exist (row0 < rows)
  __device__ __forceinline__ void issue(const Bf16* base, long long ld, int row0, int rows, uint16_t* tile) const {
    constexpr int kTurn = W == 1 && D == 128 ? 1 : W == 1 && D == 64 ? 2 : 0;  // a step of RPI rows in the permutation
    const int wv = W == 1 ? 0 : gq_wave();
    if (row0 + NR <= rows) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        gq_dma16(base + (row0 + W * RPI * i) * ld, offset + (chunk ^ (16u * (kTurn * i & 3))), tile + (W * i + wv) * 512);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int over = max(0, row0 + row + W * RPI * i - (rows - 1));  // rows past the last
        gq_dma16(base + row0 * ld, offset + (chunk ^ (16u * (kTurn * i & 3))) + (uint32_t)((W * RPI * i - over) * ld) * 2,
                 tile + (W * i + wv) * 512);
      }
    }
  }
};
// whether a tensor's rows can be fetched so: ld counted in values
inline bool gq_dma_fits(const void* p, long long ld) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0 && ld < (1 << 22);
}

// Four consecutive values of a row from column d on, n columns in all.
template <typename T>
__device__ __forceinline__ void gq_store4(T* row, int d, int n, const float (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    store_piece(row, d, n, v);
  } else {
    struct __attribute__((packed, aligned(2))) Two {
      uint32_t w[2];
    };
    if (d + 4 <= n) {
      *reinterpret_cast<Two*>(row + d) = Two{{bf16_round2(v[0], v[1]), bf16_round2(v[2], v[3])}};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (d + i < n) from_f32(row + d + i, v[i]);
    }
  }
}

// Parts joined: out[row][col] (row stride ld) = the sum of `parts` fp32 arrays [rows][cols] in order.
template <typename T>
int gqa_join_launch(int parts, size_t rows, int cols, const float* part, T* out, long long ld, hipStream_t s);

int gqa_check(const char* fn, const talos_gqa_cfg* cfg, const float* bias, const void* q, long long ld_q, const void* k,
              long long ld_k, const void* v, long long ld_v, const void* o, long long ld_o, const float* lse);
GqaArgs gqa_args(const talos_gqa_cfg* cfg, const int32_t* q_lens, const int32_t* k_lens, const float* bias, const void* q,
                 long long ld_q, const void* k, long long ld_k, const void* v, long long ld_v);

}  // namespace talos
