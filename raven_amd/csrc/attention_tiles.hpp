// attention_tiles.hpp — what the training kernels of attention share (attention_train.hip,
// attention_grad.hip): operands [batch, heads, length, dim], tiles of their rows in LDS, and the two
// kinds of products that all of them are made of.
//
// A wave has 32 columns (queries, in the gradient of keys and values keys), whose vectors are its own
// and stay in registers; rows (of the other kind) come through LDS, 32 at a time. With 32x32 matrix
// instructions
//   scores    rows x columns   = rows . columns^T     a lane has 16 rows of one column
//   results   dim x columns   += rows^T . weights     weights: function of the scores, rows x columns
// the scores' layout is the one that the second product takes its weights in: nothing goes through LDS on the
// way, and what belongs to a column is a value of a lane. A contraction may number its terms as it likes if
// both operands do, so the rows of weights stay where the first product left them (rows 4 g .. 4 g + 3 of
// every eight, g the half of the wave). rows^T is read from the same LDS tile by the transposing load (16-bit
// elements) or element by element (float32, whose matrix instruction takes one a lane).
#pragma once

#include "gemm_tile.hpp"
#include "nxh_common.hpp"

namespace {

using gemm_tile::f32x16;
using gemm_tile::lds_s16x4;
using gemm_tile::s16x4;
using gemm_tile::V16;

constexpr float LOG2E = 0x1.715476p+0f, LN2 = 0x1.62e43p-1f;
constexpr float INF = __builtin_inff();

struct HeadOperand {
  const char *base;
  int64_t batch, head, row;  // strides, elements
  int direct;                // rows are whole 16-byte units on 16-byte addresses: they may go to LDS past the registers
};
struct AttentionArgs {
  HeadOperand q, k, v, out, g, dq, dk, dv;
  HeadOperand mask;      // base null: none
  int64_t mask_col;
  HeadOperand lse;       // row: of one value each
  const int32_t *lengths;  // null: none
  int64_t lengths_step;
  float *rows;     // what each row's exponents and differences take, [batch, heads][rows_pitch][2]
  int rows_pitch;
  float *partial;  // parts' dk and dv, [parts][batch, kv_heads, sk][2][dim]; null: one part
  int parts;
  int batch, heads, kv_heads, sq, sk, dim, tiles;
  int causal, shift;  // causal: query i sees keys j <= i + shift
  float scale, c2;    // c2 = scale log2(e)
};

template <class EL>
__device__ __forceinline__ const typename EL::S *rows_of(const HeadOperand &o, int b, int h) {
  return reinterpret_cast<const typename EL::S *>(o.base) + (int64_t)b * o.batch + (int64_t)h * o.head;
}
// The keys that a sequence has.
__device__ __forceinline__ int keys_of(const AttentionArgs &a, int b) {
  if (!a.lengths) return a.sk;
  const int n = a.lengths[(int64_t)b * a.lengths_step];
  return n < 0 ? 0 : n < a.sk ? n : a.sk;
}

// Two neighbours rounded to nearest, `lo` in the low half.
template <class EL>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (EL::BF16) return f32x2_to_bf16x2(lo, hi);
  else {
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
    asm("" : "+v"(lo), "+v"(hi));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{lo, hi}, f16x2_t));
  }
}
template <class EL>
__device__ __forceinline__ void unpack2(uint32_t w, float &lo, float &hi) {
  if constexpr (EL::BF16) {
    lo = u2f(w << 16);
    hi = u2f(w & 0xffff0000u);
  } else {
    lo = (float)__builtin_bit_cast(_Float16, (uint16_t)(w & 0xffffu));
    hi = (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
  }
}
// The other half's value of the same column.
__device__ __forceinline__ float other_half(float v) {
  const uint32_t u = f2u(v);
  const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return u2f((threadIdx.x & 32) ? p[0] : p[1]);
}

// 16 bytes of a row from element c on, zeros past its end. A vector needs no more than an element's alignment.
template <class EL>
__device__ __forceinline__ V16 load_part(const typename EL::S *p, int left) {
  using S = typename EL::S;
  V16 w = {0, 0, 0, 0};
  if (left >= EL::VE) {
    __builtin_memcpy(&w, p, 16);
  } else {
    S e[EL::VE];
#pragma unroll
    for (int j = 0; j < EL::VE; j++) e[j] = j < left ? p[j] : S{};
    __builtin_memcpy(&w, e, 16);
  }
  return w;
}

// ── tiles in LDS ────────────────────────────────────────────────────────────
typedef __attribute__((address_space(3))) V16 lds_V16;
typedef __attribute__((address_space(3))) float lds_float;
typedef __attribute__((address_space(3))) gemm_tile::f32x4 lds_f32x4;
// What lies at an LDS address.
template <class P>
__device__ __forceinline__ P *at_lds(uint32_t address) {
  return reinterpret_cast<P *>((uintptr_t)address);
}
__device__ __forceinline__ uint32_t lds_address(void *p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)p; }

// Each lane's 16 (4) bytes at `base` + its offset go to consecutive LDS addresses from `lds` on. m0 carries the LDS address; the
// compiler treats it as reserved and writes it in front of each of its own uses.
__device__ __forceinline__ void load_to_lds16(const void *base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void load_to_lds4(const void *base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}
// Waits for all loads of this wave but the last N, and for its LDS accesses, then for the block's other waves.
template <int N>
__device__ __forceinline__ void meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// ROWS rows of DP elements (the head's, and zeros), brought by WAVES waves. A load to LDS fills 1 KiB without gaps, so conflicts of
// banks are avoided by choosing which 16 bytes of a row lie where: unit u of row r at u ^ turn(r). Sixteen rows' units at one
// place, and four rows' four units that half a wave of a transposing load reads, then lie in all 64 banks.
template <class EL, int DP, int ROWS, int WAVES>
struct Tile {
  using S = typename EL::S;
  static constexpr int UNITS = DP / EL::VE, ROW = DP * (int)sizeof(S), SIZE = ROWS * ROW;  // units of a row; bytes
  static constexpr int LOADS = ROWS * UNITS / 64, LPW = (LOADS + WAVES - 1) / WAVES;       // of a tile, and of a wave that has any
  static_assert(LOADS * 64 == ROWS * UNITS && LOADS % LPW == 0, "whole loads, the same number each");
  uint32_t off[LPW];  // bytes from the tile's first row
  int wave;           // of those that bring this tile; none where it is LOADS / LPW or more

  __device__ __forceinline__ static int turn(int r) {
    if constexpr (UNITS % 16 == 0 && !(EL::F32 && UNITS == 32)) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (UNITS == 32) return r & 15;
    else if constexpr (UNITS == 24) return (r >> 1) & 7;
    else if constexpr (UNITS == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else return (r >> 2) & 3;
  }
  __device__ __forceinline__ void begin(int w, int64_t row) {
    wave = w;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < LPW; i++) {
      const int u = (wave * LPW + i) * 64 + lane, r = u / UNITS;
      off[i] = (uint32_t)r * (uint32_t)row * (uint32_t)sizeof(S) + (uint32_t)((u % UNITS) ^ turn(r)) * 16u;
    }
  }
  // Units past the head's end, which loads leave as they are, in all of a tile's memory.
  __device__ __forceinline__ void clear(uint32_t tile, int dim) const {
    if (dim == DP || wave >= LOADS / LPW) return;
#pragma unroll
    for (int i = 0; i < LPW; i++) *at_lds<lds_V16>(tile + ((wave * LPW + i) * 64 + (threadIdx.x & 63)) * 16) = V16{0, 0, 0, 0};
  }
  // The rows from `first` on, of which `left` exist. Whole tiles go past the registers and arrive by meet(); others are there once
  // this returns.
  __device__ __forceinline__ void fetch(const S *first, int left, const HeadOperand &o, int dim, uint32_t tile) const {
    if (wave >= LOADS / LPW) return;
    const int lane = threadIdx.x & 63;
    const uint32_t to = tile + (uint32_t)wave * LPW * 1024u;
    if (left >= ROWS && o.direct) {
#pragma unroll
      for (int i = 0; i < LPW; i++) {
        if (dim == DP) {
          load_to_lds16(first, off[i], to + i * 1024);
        } else {
          const int u = (wave * LPW + i) * 64 + lane;
          if (((u % UNITS) ^ turn(u / UNITS)) * EL::VE < dim) load_to_lds16(first, off[i], to + i * 1024);
        }
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < LPW; i++) {
      const int u = (wave * LPW + i) * 64 + lane, r = u / UNITS, c = ((u % UNITS) ^ turn(r)) * EL::VE;
      V16 w = {0, 0, 0, 0};
      if (r < left && c < dim) w = load_part<EL>(reinterpret_cast<const S *>(reinterpret_cast<const char *>(first) + off[i]), dim - c);
      *at_lds<lds_V16>(to + (i * 64 + lane) * 16) = w;
    }
  }
};

// A column's own vectors: for step s of a product over the dim, elements 2 VE s + VE g onwards.
template <class EL, int DP>
struct Column {
  static constexpr int STEPS = DP / (2 * EL::VE);
  V16 f[STEPS];
  __device__ __forceinline__ void load(const typename EL::S *row, bool there, int dim) {
    const int g = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
      const int c = (2 * s + g) * EL::VE;
      f[s] = V16{0, 0, 0, 0};
      if (there && c < dim) f[s] = load_part<EL>(row + c, dim - c);
    }
  }
  // The lane's part of the product with another column of the same kind.
  __device__ __forceinline__ float dot(const Column &o) const {
    float sum = 0.0f;
#pragma unroll
    for (int s = 0; s < STEPS; s++)
#pragma unroll
      for (int w = 0; w < 4; w++) {
        if constexpr (EL::F32) {
          sum = __builtin_fmaf(u2f(f[s][w]), u2f(o.f[s][w]), sum);
        } else {
          float x0, x1, y0, y1;
          unpack2<EL>(f[s][w], x0, x1);
          unpack2<EL>(o.f[s][w], y0, y1);
          sum = __builtin_fmaf(x1, y1, __builtin_fmaf(x0, y0, sum));
        }
      }
    return sum;
  }
};

// What stands before it is issued before what stands behind. The compiler keeps registers free by reading from LDS right in front of
// each use, and each matrix instruction then waits out a read's latency: all of a product's reads are issued first.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

// Where a lane reads in a tile: its row's vectors, which a scores() takes, and the elements that an add() takes. The places of a
// tile's units differ by turns, which stay inside groups of four, eight or sixteen: a few addresses, made once for a stage,
// and constants beside them.
template <class T, class EL>
struct Places {
  static constexpr int GROUP = T::UNITS % 16 == 0 ? 16 : T::UNITS % 8 == 0 ? 8 : 4;
  static constexpr int VECTORS = GROUP / 2, ELEMENTS = EL::F32 ? (GROUP < 8 ? GROUP : 8) : GROUP / 2;
  uint32_t vector[VECTORS], element[ELEMENTS];
  __device__ __forceinline__ void begin() {
    const int lane = threadIdx.x & 63, r = lane & 31, g = lane >> 5;
#pragma unroll
    for (int i = 0; i < VECTORS; i++) vector[i] = (uint32_t)(r * T::ROW + (g ^ T::turn(r) ^ (2 * i)) * 16);
    if constexpr (EL::F32) {
      // row 8 (e / 4) + 4 g + e % 4, unit 8 t + c / 4: turn(row) = turn(4 g) ^ turn(8 (e / 4) + e % 4)
#pragma unroll
      for (int i = 0; i < ELEMENTS; i++) element[i] = (uint32_t)(4 * g * T::ROW + ((r >> 2) ^ T::turn(4 * g) ^ i) * 16 + (lane & 3) * 4);
    } else {
      // the transposing load: sixteen lanes read 4 rows of 16 elements, lane i eight bytes of row i / 4, and get column i's four
      const int j = (lane & 15) >> 2, b = (lane >> 4) & 1, c = (lane & 3) >> 1;
#pragma unroll
      for (int i = 0; i < ELEMENTS; i++)  // unit 2 b + c, and those that 4 t and 8 rows on (2) turn it to
        element[i] = (uint32_t)((4 * g + j) * T::ROW + ((2 * b + c) ^ T::turn(4 * g + j) ^ (2 * i)) * 16 + (lane & 1) * 8);
    }
  }
  __device__ __forceinline__ Places in(uint32_t stage) const {
    Places p;
#pragma unroll
    for (int i = 0; i < VECTORS; i++) {
      p.vector[i] = vector[i] + stage;
      asm("" : "+v"(p.vector[i]));  // (what is added to it is the instruction's offset)
    }
#pragma unroll
    for (int i = 0; i < ELEMENTS; i++) {
      p.element[i] = element[i] + stage;
      asm("" : "+v"(p.element[i]));
    }
    return p;
  }
};

// Elements of 32 rows as scores() takes them: row lane % 32. OFFSET: of the first row in a stage, a multiple of 32 of a tile's.
template <class T, class EL, int DP>
struct RowVectors {
  static constexpr int STEPS = DP / (2 * EL::VE);
  V16 f[STEPS];
  template <int OFFSET>
  __device__ __forceinline__ void load(const Places<T, EL> &p) {
    constexpr int GROUP = Places<T, EL>::GROUP;
#pragma unroll
    for (int s = 0; s < STEPS; s++) f[s] = *at_lds<const lds_V16>(p.vector[(2 * s) % GROUP / 2] + (uint32_t)((2 * s) / GROUP * GROUP * 16 + OFFSET));
  }
  // acc[e] += row (e / 4) * 8 + g * 4 + e % 4 . this lane's column
  __device__ __forceinline__ void scores(f32x16 &acc, const Column<EL, DP> &column) const {
#pragma unroll
    for (int s = 0; s < STEPS; s++) gemm_tile::mfma_step<EL>(acc, f[s], column.f[s]);
  }
};

// Weights of 32 rows and this lane's column, as the second product takes them: rounded to the operands' type, which its
// matrix instruction wants (float32 as they are).
template <class EL>
struct Weights {
  uint32_t w[8];
  __device__ __forceinline__ void set(const f32x16 &x) {
#pragma unroll
    for (int e = 0; e < 16; e += 2) w[e >> 1] = pack2<EL>(x[e], x[e + 1]);
  }
};
template <>
struct Weights<gemm_tile::ElF32> {
  f32x16 w;
  __device__ __forceinline__ void set(const f32x16 &x) { w = x; }
};

// Elements of 32 rows as the second product takes them: acc[t][e] += sum over the rows of element 32 t + (e / 4) * 8 + g * 4 +
// e % 4 of a row times its weight for this lane's column. 16-bit elements are read ahead; float32's instructions take longer than a read.
template <class T, class EL, int OT>
struct RowElements {
  V16 f[2 * OT];
  template <int OFFSET>
  __device__ __forceinline__ void load(const Places<T, EL> &p) {
    constexpr int GROUP = Places<T, EL>::GROUP;
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
      for (int t = 0; t < OT; t++) {
        const int i = (4 * t) % GROUP / 2, at = (4 * t) / GROUP * GROUP * 16 + 16 * s * T::ROW + OFFSET;
        typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(at_lds<lds_s16x4>(p.element[i] + (uint32_t)at)));
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(at_lds<lds_s16x4>(p.element[i ^ 1] + (uint32_t)(at + 8 * T::ROW))));
        f[s * OT + t] = V16{lo[0], lo[1], hi[0], hi[1]};
      }
  }
  __device__ __forceinline__ void add(f32x16 (&acc)[OT], const Weights<EL> &p) const {
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
      for (int t = 0; t < OT; t++)
        gemm_tile::mfma_step<EL>(acc[t], f[s * OT + t], V16{p.w[4 * s], p.w[4 * s + 1], p.w[4 * s + 2], p.w[4 * s + 3]});
  }
};
template <class T, int OT>
struct RowElements<T, gemm_tile::ElF32, OT> {
  const Places<T, gemm_tile::ElF32> *places;
  uint32_t offset;
  template <int OFFSET>
  __device__ __forceinline__ void load(const Places<T, gemm_tile::ElF32> &p) { places = &p, offset = OFFSET; }
  __device__ __forceinline__ void add(f32x16 (&acc)[OT], const Weights<gemm_tile::ElF32> &p) const {
    float f[2][OT];  // a row's elements are read while the row before is multiplied
    auto load = [&](int e) {
      const int r = (e >> 2) * 8 + (e & 3), turned = T::turn(r);
#pragma unroll
      for (int t = 0; t < OT; t++)
        f[e & 1][t] = *at_lds<const lds_float>(places->element[turned & 7] + (uint32_t)(((8 * t) ^ (turned & ~7)) * 16 + r * T::ROW) + offset);
    };
    load(0);
#pragma unroll
    for (int e = 0; e < 16; e++) {
      in_order();
      if (e < 15) load(e + 1);
#pragma unroll
      for (int t = 0; t < OT; t++) acc[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(f[e & 1][t], p.w[e], acc[t], 0, 0, 0);
    }
  }
};

// Two products of 32 rows each, of tiles that lie side by side: a += rows . ca, b += rows T::SIZE further on . cb. A few steps' rows
// are read while the steps before are multiplied. float32 leaves out steps past the head's end, whose instructions are slow.
template <class T, int OFFSET, class EL, int DP>
__device__ __forceinline__ void two_scores(f32x16 &a, const Column<EL, DP> &ca, f32x16 &b, const Column<EL, DP> &cb, const Places<T, EL> &p, int dim) {
  constexpr int STEPS = DP / (2 * EL::VE), CHUNK = EL::F32 ? 2 : STEPS % 4 == 0 ? 4 : STEPS < 4 ? STEPS : 3, CHUNKS = STEPS / CHUNK, GROUP = Places<T, EL>::GROUP;
  static_assert(CHUNKS * CHUNK == STEPS, "whole chunks");
  V16 f[2][CHUNK];
  auto load = [&](int i) {
#pragma unroll
    for (int k = 0; k < CHUNK; k++) {
      const int s = i % CHUNKS * CHUNK + k;
      f[i & 1][k] = *at_lds<const lds_V16>(p.vector[(2 * s) % GROUP / 2] + (uint32_t)((2 * s) / GROUP * GROUP * 16 + OFFSET + i / CHUNKS * T::SIZE));
    }
  };
  load(0);
#pragma unroll
  for (int i = 0; i < 2 * CHUNKS; i++) {
    in_order();
    if (i + 1 < 2 * CHUNKS) load(i + 1);
    if (EL::F32 && i % CHUNKS * CHUNK * 2 * EL::VE >= dim) continue;
#pragma unroll
    for (int k = 0; k < CHUNK; k++) {
      const int s = i % CHUNKS * CHUNK + k;
      if (i < CHUNKS) gemm_tile::mfma_step<EL>(a, f[i & 1][k], ca.f[s]);
      else gemm_tile::mfma_step<EL>(b, f[i & 1][k], cb.f[s]);
    }
  }
}

// Results of a lane's column, times `factor`, to its row.
template <class EL, int DP>
__device__ __forceinline__ void store_column(typename EL::S *row, const f32x16 (&acc)[DP / 32], float factor, int dim) {
  using S = typename EL::S;
  const int g = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int t = 0; t < DP / 32; t++)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int d = t * 32 + (e >> 2) * 8 + g * 4;
      S x[4];
      if constexpr (EL::F32) {
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = acc[t][e + j] * factor;
      } else {
        const uint32_t w[2] = {pack2<EL>(acc[t][e] * factor, acc[t][e + 1] * factor), pack2<EL>(acc[t][e + 2] * factor, acc[t][e + 3] * factor)};
        __builtin_memcpy(x, w, 8);
      }
      if (d + 4 <= dim) {
        __builtin_memcpy(row + d, x, sizeof x);
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (d + j < dim) row[d + j] = x[j];
      }
    }
}

// Bits e of the 16 elements a lane has of 32 rows for which row (e / 4) * 8 + e % 4 is at least `from` (of the lane's own, less 4 g).
__device__ __forceinline__ uint32_t rows_from(int from) {
  const int q = from >> 3, r = from & 7;  // the first `from` rows: 4 bits for every eight, those of the last
  const uint32_t below = from <= 0 ? 0u : from >= 32 ? 0xffffu : ((1u << (4 * q)) - 1u) | ((1u << (r < 4 ? r : 4)) - 1u) << (4 * q);
  return 0xffffu & ~below;
}
// What the mask holds for the 16 pairs of a lane: requested before the products, looked at behind them.
struct MaskBytes {
  uint32_t b[16];
  // keys j0 + (e / 4) * 8 + g * 4 + e % 4 of query qi: four neighbours are one load, of any alignment, where they lie side by side
  __device__ __forceinline__ void load_keys(const AttentionArgs &a, const uint8_t *mask, int qi, int j0) {
    const int first = j0 + ((threadIdx.x >> 5) & 1) * 4;
    const uint8_t *m = mask + (int64_t)(qi < a.sq ? qi : a.sq - 1) * a.mask.row;
    if (a.mask_col == 1 && j0 + 32 <= a.sk) {
      uint32_t four[4];
#pragma unroll
      for (int e = 0; e < 4; e++) __builtin_memcpy(&four[e], m + first + e * 8, 4);
#pragma unroll
      for (int e = 0; e < 16; e++) b[e] = (four[e >> 2] >> (8 * (e & 3))) & 0xffu;
    } else {
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const int j = first + (e >> 2) * 8 + (e & 3);
        b[e] = m[(int64_t)(j < a.sk ? j : a.sk - 1) * a.mask_col];
      }
    }
  }
  // queries i0 + (e / 4) * 8 + g * 4 + e % 4 of key kj
  __device__ __forceinline__ void load_queries(const AttentionArgs &a, const uint8_t *mask, int kj, int i0) {
    const int first = i0 + ((threadIdx.x >> 5) & 1) * 4;
    const uint8_t *m = mask + (int64_t)(kj < a.sk ? kj : a.sk - 1) * a.mask_col;
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const int i = first + (e >> 2) * 8 + (e & 3);
      b[e] = m[(int64_t)(i < a.sq ? i : a.sq - 1) * a.mask.row];
    }
  }
  __device__ __forceinline__ uint32_t kept() const {
    uint32_t k = 0;
#pragma unroll
    for (int e = 0; e < 16; e++) k |= (uint32_t)(b[e] != 0) << e;
    return k;
  }
};
// Which of those keys query qi sees, the mask aside, bit e of the result.
__device__ __forceinline__ uint32_t keys_seen(const AttentionArgs &a, int qi, int j0, int keys) {
  const int end = a.causal && qi + a.shift < keys - 1 ? qi + a.shift : keys - 1;
  return ~rows_from(end + 1 - j0 - (int)((threadIdx.x >> 5) & 1) * 4) & 0xffffu;
}

// ── host side ───────────────────────────────────────────────────────────────
int attention_operand(const char *op, const nxh_tensor *t, int dt, int64_t b, int64_t h, int64_t n, int64_t d, HeadOperand &o, bool out) {
  if (t->dtype != dt) return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
  if (t->ndim != 4 || t->shape[0] != b || t->shape[1] != h || t->shape[2] != n || t->shape[3] != d)
    return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
  for (int k = 0; k < 4 && out; k++)
    if (t->shape[k] > 1 && t->strides[k] == 0) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_OUT_ALIASED);
  if (d > 1 && t->strides[3] != 1) return nxh_fail(NXH_FAILURE, op, "rows must be contiguous");
  if (n > 1 && (t->strides[2] < 0 || t->strides[2] > (1 << 23))) return nxh_fail(NXH_FAILURE, op, "rows must follow each other within 2^23 elements");
  const int64_t es = nxh_elem_size(dt);
  o.base = (const char *)t->data + t->offset * es;
  o.batch = t->strides[0];
  o.head = t->strides[1];
  o.row = n > 1 ? t->strides[2] : 0;
  o.direct = (uintptr_t)o.base % 16 == 0 && d * es % 16 == 0 && o.row * es % 16 == 0 && (b <= 1 || o.batch * es % 16 == 0) && (h <= 1 || o.head * es % 16 == 0);
  return NXH_OK;
}

// Whether two operands that have elements begin at one address.
bool same_start(const nxh_tensor *a, const nxh_tensor *b) {
  for (const nxh_tensor *t : {a, b})
    for (int d = 0; d < t->ndim; d++)
      if (t->shape[d] == 0) return false;
  return (const char *)a->data + a->offset * (int64_t)nxh_elem_size(a->dtype) == (const char *)b->data + b->offset * (int64_t)nxh_elem_size(b->dtype);
}

// What both entry points check.
int attention_arguments(const char *op, AttentionArgs &a, const nxh_tensor *q, const nxh_tensor *k, const nxh_tensor *v, const nxh_tensor *out,
                        const nxh_tensor *lse, const nxh_tensor *lengths, const nxh_tensor *mask, double scale, int causal, bool grad) {
  int rc;
  const int dt = q->dtype;
  if (dt != NXH_BF16 && dt != NXH_F16 && dt != NXH_F32) return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
  if (q->ndim != 4 || k->ndim != 4) return nxh_fail(NXH_INVALID_ARGUMENT, op, "operands must be [batch, heads, length, dim]");
  const int64_t b = q->shape[0], h = q->shape[1], sq = q->shape[2], d = q->shape[3], hk = k->shape[1], sk = k->shape[2];
  if (hk == 0 ? h != 0 : h % hk != 0) return nxh_fail(NXH_INVALID_ARGUMENT, op, "heads must be a multiple of the heads of keys and values");
  if (!(scale >= 1e-30 && scale <= 1e30)) return nxh_fail(NXH_INVALID_ARGUMENT, op, "scale must lie in 1e-30 to 1e30");  // (a normal float32)
  if (d < 1) return nxh_fail(NXH_INVALID_ARGUMENT, op, "head dimension must not be 0");
  if (d > 128) return nxh_fail(NXH_FAILURE, op, "head dimension must be at most 128");
  if (sq > 0x3fffff00 || sk > 0x3fffff00) return nxh_fail(NXH_FAILURE, op, "more than 2^30 - 256 queries or keys");
  if ((double)b * (double)h * (double)std::max<int64_t>(1, std::max(sq, sk)) > 2147483647.0) return nxh_fail(NXH_FAILURE, op, "too many rows for one launch");
  if ((rc = attention_operand(op, q, dt, b, h, sq, d, a.q, false)) || (rc = attention_operand(op, k, dt, b, hk, sk, d, a.k, false)) ||
      (rc = attention_operand(op, v, dt, b, hk, sk, d, a.v, false)) || (rc = attention_operand(op, out, dt, b, h, sq, d, a.out, !grad)))
    return rc;
  if (lse->dtype != NXH_F32) return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
  if (lse->ndim != 3 || lse->shape[0] != b || lse->shape[1] != h || lse->shape[2] != sq) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
  for (int n = 0; n < 3 && !grad; n++)
    if (lse->shape[n] > 1 && lse->strides[n] == 0) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_OUT_ALIASED);
  a.lse = {(const char *)lse->data + lse->offset * 4, lse->strides[0], lse->strides[1], lse->strides[2], 0};
  a.lengths = nullptr;
  a.lengths_step = 0;
  if (lengths) {
    if (lengths->dtype != NXH_I32) return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
    if (lengths->ndim != 1 || lengths->shape[0] != b) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
    a.lengths = (const int32_t *)lengths->data + lengths->offset;
    a.lengths_step = lengths->strides[0];
  }
  a.mask = {nullptr, 0, 0, 0, 0};
  a.mask_col = 0;
  if (mask) {
    if (mask->dtype != NXH_BOOL) return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
    if (mask->ndim != 4 || mask->shape[0] != b || mask->shape[1] != h || mask->shape[2] != sq || mask->shape[3] != sk)
      return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
    a.mask = {(const char *)mask->data + mask->offset, mask->strides[0], mask->strides[1], mask->strides[2], 0};
    a.mask_col = mask->strides[3];
  }
  a.batch = (int)b;
  a.heads = (int)h;
  a.kv_heads = (int)hk;
  a.sq = (int)sq;
  a.sk = (int)sk;
  a.dim = (int)d;
  a.causal = causal ? 1 : 0;
  a.shift = (int)(sk - sq);
  a.scale = (float)scale;
  a.c2 = (float)(scale * 1.4426950408889634);
  a.g = a.dq = a.dk = a.dv = {nullptr, 0, 0, 0, 0};
  a.rows = a.partial = nullptr;
  a.parts = 1;
  a.tiles = 0;
  return NXH_OK;
}

}  // namespace
