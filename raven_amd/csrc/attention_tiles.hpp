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
};
struct AttentionArgs {
  HeadOperand q, k, v, out, g, dq, dk, dv;
  HeadOperand mask;      // base null: none
  int64_t mask_col;
  HeadOperand lse;       // row: of one value each
  const int32_t *lengths;  // null: none
  int64_t lengths_step;
  float *delta;    // [batch, heads, sq]
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

// A tile of ROWS rows of DP elements (the head's, and zeros) in LDS, brought by 256 threads (as many of them as divide its
// vectors) through registers. Rows are 16 bytes (128 elements of 16 bits: 48) further apart than they are long: sixteen rows'
// vectors at one place lie in different banks, and of the four rows of a transposing load no more than two in one.
template <class EL, int DP, int ROWS>
struct Tile {
  using S = typename EL::S;
  static constexpr int PITCH = DP + EL::VE * (!EL::F32 && DP == 128 ? 3 : 1), SIZE = ROWS * PITCH, VPR = DP / EL::VE, ALL = ROWS * VPR;
  static constexpr int THREADS = ALL % 256 == 0 ? 256 : ALL % 192 == 0 ? 192 : ALL, NV = ALL / THREADS;
  static_assert(THREADS <= 256 && NV * THREADS == ALL, "whole vectors a thread");
  V16 pre[NV];
  uint32_t off[NV];  // bytes from the tile's first row

  __device__ __forceinline__ static bool brings() { return THREADS == 256 || (threadIdx.x & 255) < THREADS; }
  __device__ __forceinline__ void begin(int64_t row) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int v = (int)(threadIdx.x & 255) + i * THREADS;
      off[i] = ((uint32_t)(v / VPR) * (uint32_t)row + (uint32_t)(v % VPR) * EL::VE) * (uint32_t)sizeof(S);
    }
  }
  // The rows from `first` on, of which `left` exist.
  __device__ __forceinline__ void fetch(const S *first, int left, int dim) {
    if (!brings()) return;
    const char *at = reinterpret_cast<const char *>(first);
    if (left >= ROWS && dim == DP) {
#pragma unroll
      for (int i = 0; i < NV; i++) __builtin_memcpy(&pre[i], at + off[i], 16);
      return;
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int v = (int)(threadIdx.x & 255) + i * THREADS, c = (v % VPR) * EL::VE;
      pre[i] = V16{0, 0, 0, 0};
      if (v / VPR < left && c < dim) pre[i] = load_part<EL>(reinterpret_cast<const S *>(at + off[i]), dim - c);
    }
  }
  __device__ __forceinline__ void lay(S *tile) const {
    if (!brings()) return;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int v = (int)(threadIdx.x & 255) + i * THREADS;
      *reinterpret_cast<V16 *>(tile + (v / VPR) * PITCH + (v % VPR) * EL::VE) = pre[i];
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

// acc[e] += row (e / 4) * 8 + g * 4 + e % 4 of 32 . this lane's column.
template <class EL, int DP, int PITCH>
__device__ __forceinline__ void rows_by_columns(f32x16 &acc, const typename EL::S *rows, const Column<EL, DP> &column) {
  const typename EL::S *at = rows + (threadIdx.x & 31) * PITCH + ((threadIdx.x >> 5) & 1) * EL::VE;
#pragma unroll
  for (int s = 0; s < Column<EL, DP>::STEPS; s++) {
    const V16 r = *reinterpret_cast<const V16 *>(at + s * 2 * EL::VE);
    gemm_tile::mfma_step<EL>(acc, r, column.f[s]);
  }
}

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

// acc[t][e] += sum over 32 rows of element 32 t + (e / 4) * 8 + g * 4 + e % 4 of a row times its weight for this lane's column.
template <class EL, int DP, int PITCH>
__device__ __forceinline__ void add_weighted_rows(f32x16 (&acc)[DP / 32], const typename EL::S *rows, const Weights<EL> &p) {
  const int lane = threadIdx.x & 63, g = lane >> 5;
  if constexpr (EL::F32) {
    const float *at = rows + 4 * g * PITCH + (lane & 31);
#pragma unroll
    for (int e = 0; e < 16; e++)
#pragma unroll
      for (int t = 0; t < DP / 32; t++)
        acc[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(at[((e >> 2) * 8 + (e & 3)) * PITCH + t * 32], p.w[e], acc[t], 0, 0, 0);
  } else {
    const uint16_t *at = rows + (4 * g + ((lane & 15) >> 2)) * PITCH + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
      for (int t = 0; t < DP / 32; t++) {
        const uint16_t *src = at + 16 * s * PITCH + t * 32;
        typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)src));
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(src + 8 * PITCH)));
        gemm_tile::mfma_step<EL>(acc[t], V16{lo[0], lo[1], hi[0], hi[1]}, V16{p.w[4 * s], p.w[4 * s + 1], p.w[4 * s + 2], p.w[4 * s + 3]});
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

// Which of keys j0 + (e / 4) * 8 + g * 4 + e % 4 query qi sees, bit e of the result.
__device__ __forceinline__ uint32_t keys_seen(const AttentionArgs &a, const uint8_t *mask, int qi, int j0, int keys) {
  const int g = (threadIdx.x >> 5) & 1, first = j0 + g * 4;
  const int end = a.causal && qi + a.shift < keys - 1 ? qi + a.shift : keys - 1, last = end - first;
  uint32_t seen = 0;
#pragma unroll
  for (int e = 0; e < 16; e++) seen |= (uint32_t)((e >> 2) * 8 + (e & 3) <= last) << e;
  if (!mask) return seen;
  const uint8_t *m = mask + (int64_t)(qi < a.sq ? qi : a.sq - 1) * a.mask.row;
  uint32_t kept = 0;
  if (a.mask_col == 1 && j0 + 32 <= a.sk) {  // four neighbours are one load, of any alignment
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      uint32_t four;
      __builtin_memcpy(&four, m + first + e * 2, 4);
#pragma unroll
      for (int j = 0; j < 4; j++) kept |= (uint32_t)(((four >> (8 * j)) & 0xffu) != 0) << (e + j);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const int j = first + (e >> 2) * 8 + (e & 3);
      kept |= (uint32_t)(m[(int64_t)(j < a.sk ? j : a.sk - 1) * a.mask_col] != 0) << e;
    }
  }
  return seen & kept;
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
  o.base = (const char *)t->data + t->offset * (int64_t)nxh_elem_size(dt);
  o.batch = t->strides[0];
  o.head = t->strides[1];
  o.row = n > 1 ? t->strides[2] : 0;
  return NXH_OK;
}

// Whether two operands begin at one element.
bool same_start(const nxh_tensor *a, const nxh_tensor *b) {
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
  if (!(scale > 0.0 && scale <= 1e30)) return nxh_fail(NXH_INVALID_ARGUMENT, op, "scale must be positive and at most 1e30");
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
  a.lse = {(const char *)lse->data + lse->offset * 4, lse->strides[0], lse->strides[1], lse->strides[2]};
  a.lengths = nullptr;
  a.lengths_step = 0;
  if (lengths) {
    if (lengths->dtype != NXH_I32) return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
    if (lengths->ndim != 1 || lengths->shape[0] != b) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
    a.lengths = (const int32_t *)lengths->data + lengths->offset;
    a.lengths_step = lengths->strides[0];
  }
  a.mask = {nullptr, 0, 0, 0};
  a.mask_col = 0;
  if (mask) {
    if (mask->dtype != NXH_BOOL) return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
    if (mask->ndim != 4 || mask->shape[0] != b || mask->shape[1] != h || mask->shape[2] != sq || mask->shape[3] != sk)
      return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
    a.mask = {(const char *)mask->data + mask->offset, mask->strides[0], mask->strides[1], mask->strides[2]};
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
  a.g = a.dq = a.dk = a.dv = {nullptr, 0, 0, 0};
  a.delta = a.partial = nullptr;
  a.parts = 1;
  a.tiles = 0;
  return NXH_OK;
}

}  // namespace
