// rotary.hip — nxh_rotary: positions as rotations. The first r = 2 n dimensions of a head are n pairs, pair i of a row at position s is
// turned by the angle s f_i:
//   (a, b) -> A (a cos - b sin, a sin + b cos)
// and the rest is copied. Pairs are neighbours (2 i, 2 i + 1) or halves (i, i + n). The gradient is the same call with the angles
// negated. Queries and keys, which share positions, go in one launch.
//
// Angles are float64: at position 10^6 float32 is off by 0.06. They are taken in quarter turns, s f 2 / pi, whose whole number
// chooses the quadrant; what is left, at most half a quarter, goes to float32 and its sine and cosine. A lane makes them once
// for a vector of pairs and turns that of HEADS heads, whose vectors are on their way meanwhile. Elements are
// read and written by one lane each, so a result may be its operand.
//
// What bounds it: memory, where there are many rows ([8,12 + 12,1024,64] bfloat16 12 us, 4.1 TB/s), and the making of the angles, some
// 80 instructions a pair. A wave that copies one vector and turns another takes both times, so rows' pairs come
// first and what is copied after them: [3,6 + 2,2777,80] float32, 20 of them turned, 12.4 us (with each row's vectors one after
// the other 16.1). One head a lane made each angle once a head.

#include "lane_groups.hpp"

namespace {

constexpr int HEADS = 4;  // of a lane
constexpr uint32_t ROWS = 64;

struct RotaryOperand {
  const char *in;
  char *out;  // a copy is left out where it is the operand itself
  int64_t in_batch, in_head, in_row, out_batch, out_head, out_row;
  int heads, groups;  // groups of HEADS
};
struct RotaryArgs {
  RotaryOperand x[2];
  const int32_t *positions;
  int64_t position_batch, position_row;
  const double *frequencies;
  int64_t frequency_step;
  uint32_t batch, length, vectors;  // vectors of pairs of a row, and of what is copied
  uint32_t rows, total;  // rows of groups of heads; lanes
  int pairs, pair_vectors, dim;
  int inverse;
  double amplitude;
};

__device__ __forceinline__ void turn_of(double quarters, float &cosine, float &sine) {
  const double q = __builtin_rint(quarters);
  const float rest = (float)(quarters - q);  // in quarter turns, -1/2 .. 1/2
  float s, c;
  sincospif(0.5f * rest, &s, &c);
  const int n = (int)(int64_t)(q - 4.0 * __builtin_floor(q * 0.25));
  const float a = n & 1 ? s : c, b = n & 1 ? c : s;
  cosine = n == 1 || n == 2 ? -a : a;
  sine = n >= 2 ? -b : b;
}
__device__ __forceinline__ void turn_of(double quarters, double &cosine, double &sine) {
  const double q = __builtin_rint(quarters);
  double s, c;
  sincospi(0.5 * (quarters - q), &s, &c);
  const int n = (int)(int64_t)(q - 4.0 * __builtin_floor(q * 0.25));
  const double a = n & 1 ? s : c, b = n & 1 ? c : s;
  cosine = n == 1 || n == 2 ? -a : a;
  sine = n >= 2 ? -b : b;
}

template <int DT, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  using IO = Io<DT>;
  using C = typename IO::C;
  using S = typename IO::S;
  constexpr int V = IO::V;
  const uint32_t id = blockIdx.x * 256 + threadIdx.x;
  if (id >= a.total) return;
  // Of ROWS rows first the vectors of pairs, then those that are copied: other waves'.
  const uint32_t turned = (uint32_t)a.pair_vectors, copied = a.vectors - turned, chunk = id / (ROWS * a.vectors);
  uint32_t vector = id - chunk * (ROWS * a.vectors), rest;
  if (vector < ROWS * turned) {
    rest = vector / turned;
    vector -= rest * turned;
  } else {
    vector -= ROWS * turned;
    rest = vector / copied;
    vector += turned - rest * copied;
  }
  rest += chunk * ROWS;
  if (rest >= a.rows) return;
  const uint32_t row = rest % a.length;
  rest /= a.length;
  const uint32_t b = rest % a.batch;
  int group = (int)(rest / a.batch);
  const bool second = group >= a.x[0].groups;
  if (second) group -= a.x[0].groups;
  const RotaryOperand &o = a.x[second ? 1 : 0];
  const int head = group * HEADS, heads = o.heads - head < HEADS ? o.heads - head : HEADS;
  const S *in = reinterpret_cast<const S *>(o.in) + (int64_t)b * o.in_batch + (int64_t)row * o.in_row + (int64_t)head * o.in_head;
  S *out = reinterpret_cast<S *>(o.out) + (int64_t)b * o.out_batch + (int64_t)row * o.out_row + (int64_t)head * o.out_head;

  if ((int)vector >= a.pair_vectors) {  // copied
    const int c = 2 * a.pairs + ((int)vector - a.pair_vectors) * V;
    if (c + V <= a.dim) {
      Words x[HEADS];
#pragma unroll
      for (int h = 0; h < HEADS; h++) x[h] = load_words(in + (h < heads ? h : 0) * o.in_head + c);
#pragma unroll
      for (int h = 0; h < HEADS; h++)
        if (h < heads) store_words(out + h * o.out_head + c, x[h]);
    } else {
      for (int h = 0; h < heads; h++)
        for (int j = c; j < a.dim; j++) out[h * o.out_head + j] = in[h * o.in_head + j];
    }
    return;
  }
  const int pair = (int)vector * V, there = a.pairs - pair < V ? a.pairs - pair : V;
  const int c0 = INTERLEAVED ? 2 * pair : pair, c1 = INTERLEAVED ? 2 * pair + V : pair + a.pairs;
  const bool whole = there == V;
  Words x0[HEADS], x1[HEADS];
  if (whole) {
#pragma unroll
    for (int h = 0; h < HEADS; h++) {
      const int at = h < heads ? h : 0;
      x0[h] = load_words(in + at * o.in_head + c0);
      x1[h] = load_words(in + at * o.in_head + c1);
    }
  }
  const double position = (double)a.positions[(int64_t)b * a.position_batch + (int64_t)row * a.position_row] * 0.63661977236758134308;
  C cosine[V], sine[V];
#pragma unroll
  for (int j = 0; j < V; j++) {
    turn_of(j < there ? position * a.frequencies[(int64_t)(pair + j) * a.frequency_step] : 0.0, cosine[j], sine[j]);
    cosine[j] = cosine[j] * (C)a.amplitude;
    sine[j] = sine[j] * (C)(a.inverse ? -a.amplitude : a.amplitude);
  }
  if (whole) {
#pragma unroll
    for (int h = 0; h < HEADS; h++) {
      if (h >= heads) break;
      C y0[V], y1[V];
      IO::widen(x0[h], y0);
      IO::widen(x1[h], y1);
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int j = 0; j < V; j++) {
          C &p = 2 * j < V ? y0[(2 * j) % V] : y1[(2 * j) % V], &q = 2 * j < V ? y0[(2 * j + 1) % V] : y1[(2 * j + 1) % V];
          const C s = p * cosine[j] - q * sine[j], t = p * sine[j] + q * cosine[j];
          p = s;
          q = t;
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; j++) {
          const C s = y0[j] * cosine[j] - y1[j] * sine[j], t = y0[j] * sine[j] + y1[j] * cosine[j];
          y0[j] = s;
          y1[j] = t;
        }
      }
      store_words(out + h * o.out_head + c0, IO::narrow(y0));
      store_words(out + h * o.out_head + c1, IO::narrow(y1));
    }
  } else {
    S p[HEADS][V], q[HEADS][V];
#pragma unroll
    for (int h = 0; h < HEADS; h++)
#pragma unroll
      for (int j = 0; j < V - 1; j++) {
        const int i = pair + (j < there ? j : 0), ia = INTERLEAVED ? 2 * i : i, ib = INTERLEAVED ? ia + 1 : ia + a.pairs;
        const S *from = in + (h < heads ? h : 0) * o.in_head;
        p[h][j] = from[ia];
        q[h][j] = from[ib];
      }
#pragma unroll
    for (int h = 0; h < HEADS; h++)
#pragma unroll
      for (int j = 0; j < V - 1; j++) {
        if (h >= heads || j >= there) continue;
        const int ia = INTERLEAVED ? 2 * (pair + j) : pair + j, ib = INTERLEAVED ? ia + 1 : ia + a.pairs;
        const C x = IO::ld(p[h][j]), y = IO::ld(q[h][j]);
        out[h * o.out_head + ia] = IO::st(x * cosine[j] - y * sine[j]);
        out[h * o.out_head + ib] = IO::st(x * sine[j] + y * cosine[j]);
      }
  }
}

template <int DT>
void launch(nxh_context *ctx, const RotaryArgs &a, bool interleaved) {
  const dim3 grid((a.total + 255) / 256);
  if (interleaved) hipLaunchKernelGGL((rotary_kernel<DT, true>), grid, dim3(256), 0, ctx->stream, a);
  else hipLaunchKernelGGL((rotary_kernel<DT, false>), grid, dim3(256), 0, ctx->stream, a);
}

// Whether two tensors are one view: the same elements in the same order.
bool one_view(const nxh_tensor *a, const nxh_tensor *b) {
  const int64_t es = (int64_t)nxh_elem_size(a->dtype);
  if ((const char *)a->data + a->offset * es != (const char *)b->data + b->offset * es) return false;
  for (int d = 0; d < a->ndim; d++)
    if (a->shape[d] > 1 && a->strides[d] != b->strides[d]) return false;
  return true;
}

}  // namespace

NXH_EXPORT int nxh_rotary(nxh_context *ctx, const nxh_tensor *q_out, const nxh_tensor *k_out, const nxh_tensor *q, const nxh_tensor *k,
                          const nxh_tensor *positions, const nxh_tensor *frequencies, double amplitude, int flags) {
  NXH_DEFER_TOUCH(ctx, 2, q_out, k_out, q, k, positions, frequencies);
  const char *op = "rotary";
  if (!ctx || !q_out || !q || !positions || !frequencies || (!k_out) != (!k)) return nxh_fail(NXH_INVALID_ARGUMENT, op, "null argument");
  int rc;
  for (const nxh_tensor *t : {q_out, k_out, q, k, positions, frequencies})
    if (t && (rc = nxh_check_tensor(op, t))) return rc;
  const int dt = q->dtype;
  if ((dt != NXH_F32 && dt != NXH_BF16 && dt != NXH_F16 && dt != NXH_F64) || positions->dtype != NXH_I32 || frequencies->dtype != NXH_F64)
    return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
  if (flags & ~3) return nxh_fail(NXH_INVALID_ARGUMENT, op, "unknown flag");
  if (!(amplitude - amplitude == 0.0)) return nxh_fail(NXH_INVALID_ARGUMENT, op, "amplitude must be finite");
  RotaryArgs a;
  a.x[1] = {};
  bool in_place = true;
  const nxh_tensor *ins[] = {q, k}, *outs[] = {q_out, k_out};
  for (int i = 0; i < 2; i++) {
    const nxh_tensor *x = ins[i], *y = outs[i];
    if (!x) continue;
    if (x->ndim != 4) return nxh_fail(NXH_INVALID_ARGUMENT, op, "operands must be [batch, heads, length, dim]");
    if (x->dtype != dt || y->dtype != dt) return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
    if (!nxh_same_shape(x, y) || x->shape[0] != q->shape[0] || x->shape[2] != q->shape[2] || x->shape[3] != q->shape[3])
      return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
    for (int d = 0; d < 4; d++)
      if (y->shape[d] > 1 && y->strides[d] == 0) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_OUT_ALIASED);
    if (x->shape[3] > 1 && (x->strides[3] != 1 || y->strides[3] != 1)) return nxh_fail(NXH_FAILURE, op, "rows must be contiguous");
    const int64_t es = nxh_elem_size(dt);
    if (x->shape[1] > 0x7ffffff0) return nxh_fail(NXH_FAILURE, op, "extent exceeds 32 bits");
    a.x[i] = {(const char *)x->data + x->offset * es, (char *)y->data + y->offset * es, x->strides[0], x->strides[1], x->strides[2],
              y->strides[0], y->strides[1], y->strides[2], (int)x->shape[1], (int)((x->shape[1] + HEADS - 1) / HEADS)};
    in_place = in_place && one_view(x, y);
  }
  if (k && a.x[0].out == a.x[1].out && a.x[0].heads > 0 && a.x[1].heads > 0 && q->shape[0] > 0 && q->shape[2] > 0 && q->shape[3] > 0)
    return nxh_fail(NXH_INVALID_ARGUMENT, op, "two results in one place");
  const int64_t batch = q->shape[0], length = q->shape[2], dim = q->shape[3];
  if (positions->ndim != 2 || positions->shape[0] != batch || positions->shape[1] != length || frequencies->ndim != 1)
    return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
  const int64_t pairs = frequencies->shape[0];
  if (2 * pairs > dim) return nxh_fail(NXH_INVALID_ARGUMENT, op, "more frequencies than pairs of dimensions");
  if (dim > ((int64_t)1 << 24)) return nxh_fail(NXH_FAILURE, op, "rows longer than 2^24 elements");
  const int v = (int)(16 / nxh_elem_size(dt));
  a.pairs = (int)pairs;
  a.dim = (int)dim;
  a.pair_vectors = (int)((pairs + v - 1) / v);
  const int64_t vectors = a.pair_vectors + (in_place ? 0 : (dim - 2 * pairs + v - 1) / v), groups = (int64_t)a.x[0].groups + a.x[1].groups;
  if (batch == 0 || length == 0 || vectors == 0 || groups == 0) return NXH_OK;
  if (((double)batch * (double)length * (double)groups + ROWS) * (double)vectors > 4294967040.0) return nxh_fail(NXH_FAILURE, op, "too many rows for one launch");
  a.batch = (uint32_t)batch;
  a.length = (uint32_t)length;
  a.vectors = (uint32_t)vectors;
  a.rows = (uint32_t)(batch * length * groups);
  a.total = (a.rows + ROWS - 1) / ROWS * ROWS * a.vectors;
  a.positions = (const int32_t *)positions->data + positions->offset;
  a.position_batch = positions->strides[0];
  a.position_row = positions->strides[1];
  a.frequencies = (const double *)frequencies->data + frequencies->offset;
  a.frequency_step = frequencies->strides[0];
  a.inverse = flags & 2;
  a.amplitude = amplitude;
  std::lock_guard<std::mutex> guard(ctx->mu);
  NXH_HIP(op, hipSetDevice(ctx->device));
  nxh_set_path("rotary");
  const bool interleaved = flags & 1;
  if (dt == NXH_F32) launch<NXH_F32>(ctx, a, interleaved);
  else if (dt == NXH_BF16) launch<NXH_BF16>(ctx, a, interleaved);
  else if (dt == NXH_F16) launch<NXH_F16>(ctx, a, interleaved);
  else launch<NXH_F64>(ctx, a, interleaved);
  NXH_HIP(op, hipGetLastError());
  return NXH_OK;
}
