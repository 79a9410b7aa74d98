// rows.hpp — what the kernels over rows of a tensor share (rowfuse.hip, layer_norm.hip,
// layer_norm_grad.hip, log_probs.hip): the rows of operands that have a layout of their own,
// and the host's checks of them. A row is the last axis.
#pragma once

#include <initializer_list>

#include "nxh_common.hpp"

namespace {

constexpr int ROW_MAXD = 8;
constexpr int64_t ROW_MAX = (int64_t)1 << 24;  // the longest row at all (float32 counts it exactly)

struct RowGeom {
  int64_t rows;
  int n, nouter;
  uint32_t oshape[ROW_MAXD];
};
struct RowOperand {
  const char *base;
  int64_t stride[ROW_MAXD];  // per outer dim, elements
};

// Where row `row` begins in each of K operands, in elements.
template <int K>
__device__ __forceinline__ void row_starts(const RowGeom &g, uint32_t row, const RowOperand (&operands)[K], int64_t (&at)[K]) {
#pragma unroll
  for (int k = 0; k < K; k++) at[k] = 0;
  uint32_t r = row;
  for (int d = g.nouter - 1; d > 0; d--) {  // (the host has merged what composes: usually one dim and no division)
    const uint32_t q = r / g.oshape[d], i = r - q * g.oshape[d];
    r = q;
#pragma unroll
    for (int k = 0; k < K; k++) at[k] += (int64_t)i * operands[k].stride[d];
  }
#pragma unroll
  for (int k = 0; k < K; k++) at[k] += (int64_t)r * operands[k].stride[0];  // (no outer dim: the strides are 0)
}

// ── host side ───────────────────────────────────────────────────────────────
bool float_dtype_ok(int dt) { return dt == NXH_F32 || dt == NXH_F64 || dt == NXH_BF16 || dt == NXH_F16; }

// Fills the row geometry from `x` (rows = product of the outer extents).
int row_geometry(const char *op, const nxh_tensor *x, RowGeom &g) {
  if (x->ndim < 1) return nxh_fail(NXH_INVALID_ARGUMENT, op, "input must not be a scalar");
  if (x->ndim - 1 > ROW_MAXD) return nxh_fail(NXH_FAILURE, op, "more than 8 outer dimensions");
  if (x->shape[x->ndim - 1] > ROW_MAX) return nxh_fail(NXH_FAILURE, op, "rows longer than 2^24 elements");
  g.n = (int)x->shape[x->ndim - 1];
  g.nouter = x->ndim - 1;
  g.rows = 1;
  for (int d = 0; d < g.nouter; d++) {
    if (x->shape[d] > 0xffffffffLL) return nxh_fail(NXH_FAILURE, op, "extent exceeds 32 bits");
    g.oshape[d] = (uint32_t)x->shape[d];
    g.rows *= x->shape[d];
  }
  return NXH_OK;
}
void row_operand(const nxh_tensor *t, RowOperand &o) {
  o.base = t ? (const char *)t->data + t->offset * (int64_t)nxh_elem_size(t->dtype) : nullptr;
  for (int d = 0; d < ROW_MAXD; d++) o.stride[d] = (t && d < t->ndim - 1) ? t->strides[d] : 0;
}
// Outer dims that compose on every operand (stride[d - 1] == stride[d] * extent[d], a broadcast
// with both strides 0 included) become one: contiguous rows end up with a single outer dim.
void merge_outer_dims(RowGeom &g, std::initializer_list<RowOperand *> ops) {
  int n = g.nouter;
  for (int d = n - 1; d > 0; d--) {
    bool composes = true;
    for (RowOperand *o : ops) composes = composes && o->stride[d - 1] == o->stride[d] * (int64_t)g.oshape[d];
    if (!composes || (uint64_t)g.oshape[d - 1] * g.oshape[d] > 0xffffffffULL) continue;
    g.oshape[d - 1] *= g.oshape[d];
    for (RowOperand *o : ops) o->stride[d - 1] = o->stride[d];
    for (int e = d; e + 1 < n; e++) {
      g.oshape[e] = g.oshape[e + 1];
      for (RowOperand *o : ops) o->stride[e] = o->stride[e + 1];
    }
    n--;
  }
  g.nouter = n;
}
// A row operand can be moved V elements at a time when its rows are contiguous
// and every row starts on a V-element boundary.
bool rows_vector_ok(const nxh_tensor *t, int v) {
  const int es = (int)nxh_elem_size(t->dtype);
  if ((((uintptr_t)t->data + t->offset * es) % (uintptr_t)(es * v)) != 0) return false;
  for (int d = 0; d < t->ndim - 1; d++)
    if (t->shape[d] > 1 && t->strides[d] % v != 0) return false;
  return true;
}
// Rows of a and b are off their V-element boundaries by the same amount, row by row: the
// long-row kernels then peel the same head and tail from both.
bool rows_congruent(const nxh_tensor *a, const nxh_tensor *b, int v) {
  const uintptr_t ea = (uintptr_t)a->data / nxh_elem_size(a->dtype) + (uintptr_t)a->offset;
  const uintptr_t eb = (uintptr_t)b->data / nxh_elem_size(b->dtype) + (uintptr_t)b->offset;
  if ((uintptr_t)a->data % nxh_elem_size(a->dtype) || (uintptr_t)b->data % nxh_elem_size(b->dtype)) return false;
  if (ea % v != eb % v) return false;
  for (int d = 0; d < a->ndim - 1; d++)
    if (a->shape[d] > 1 && ((a->strides[d] - b->strides[d]) % v) != 0) return false;
  return true;
}
int same_shape(const char *op, const nxh_tensor *a, const nxh_tensor *b) {
  if (a->ndim != b->ndim) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
  for (int d = 0; d < a->ndim; d++)
    if (a->shape[d] != b->shape[d]) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
  return NXH_OK;
}
int out_rows_ok(const char *op, const nxh_tensor *out) {
  for (int d = 0; d < out->ndim; d++)
    if (out->shape[d] > 1 && out->strides[d] == 0) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_OUT_ALIASED);
  return NXH_OK;
}

// ── rows with a value each (statistics, tokens, upstream gradients) ─────────
// row_geometry for launches that number their rows in 32 bits.
int rows_geometry(const char *op, const nxh_tensor *x, RowGeom &g) {
  bool none = false;
  double rows = 1;  // (extents of broadcast dims have products past 64 bits)
  for (int d = 0; d + 1 < x->ndim; d++) {
    none = none || x->shape[d] == 0;
    rows *= (double)x->shape[d];
  }
  if (!none && rows > 2147483647.0) return nxh_fail(NXH_FAILURE, op, "too many rows for one launch");
  return row_geometry(op, x, g);
}
// What sums and statistics of a dtype are held and given out in.
int statistics_dtype(int dt) { return dt == NXH_F64 ? NXH_F64 : NXH_F32; }
// A tensor with one value per row of x.
int row_values_ok(const char *op, const nxh_tensor *t, const nxh_tensor *x, int dtype) {
  if (t->dtype != dtype) return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
  if (t->ndim != x->ndim - 1) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
  for (int d = 0; d < t->ndim; d++)
    if (t->shape[d] != x->shape[d]) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
  return NXH_OK;
}
void row_value_operand(const nxh_tensor *t, RowOperand &o) {
  o.base = t ? (const char *)t->data + t->offset * (int64_t)nxh_elem_size(t->dtype) : nullptr;
  for (int d = 0; d < ROW_MAXD; d++) o.stride[d] = (t && d < t->ndim) ? t->strides[d] : 0;
}
// A contiguous vector of a row's length.
int row_vector_ok(const char *op, const nxh_tensor *t, int n) {
  if (t->ndim != 1 || t->shape[0] != n) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
  if (n > 1 && t->strides[0] != 1) return nxh_fail(NXH_FAILURE, op, "rows must be contiguous");
  return NXH_OK;
}
// Whether two tensors are one view: the same elements in the same order.
bool same_view(const nxh_tensor *a, const nxh_tensor *b) {
  if (a->dtype != b->dtype || a->ndim != b->ndim) return false;
  const int64_t es = (int64_t)nxh_elem_size(a->dtype);
  if ((const char *)a->data + a->offset * es != (const char *)b->data + b->offset * es) return false;
  for (int d = 0; d < a->ndim; d++)
    if (a->shape[d] != b->shape[d] || (a->shape[d] > 1 && a->strides[d] != b->strides[d])) return false;
  return true;
}
bool unit_stride(const nxh_tensor *t) { return t->shape[t->ndim - 1] <= 1 || t->strides[t->ndim - 1] == 1; }

}  // namespace
