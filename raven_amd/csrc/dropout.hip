// dropout.hip — nxh_dropout: out = residual + (u >= cut ? x * scale : 0) with random bits that are
// made where they are used. Element i (its row-major position in x's shape) belongs to block i / 4 of
// Threefry-2x32-20 under the key; its u are 16 of the block's 64 bits: the low and the high half of the
// first word, then of the second. cut = round(65536 rate) and scale = 65536 / (65536 - cut), so what is
// kept has x as its mean exactly. The mask is never stored: the transposed step is the same call on the
// gradient, with the same key and rate.
//
// x (and the residual) in, out out. A block of the generator is some 75 vector instructions; 32 bits for
// each element, two to a block, would have made them the bound for 16-bit dtypes, where four to a block
// leave both at about the same. A rate is then off by at most 2^-17, which scale accounts for. [98304,1024]
// bfloat16 69 us (5.8 TB/s), [8192,768] with its residual 7.0 us (5.4 TB/s).

#include <cmath>

#include "lane_groups.hpp"
#include "threefry.hpp"

namespace {

constexpr int DROP_MAXD = NXH_MAX_NDIM;
constexpr int64_t DROP_BLOCKS = 1 << 20;  // of a launch, which numbers its lanes in 32 bits; they go on with the rest
struct DropoutArgs {
  const char *x, *residual;  // residual: null for none
  char *out;
  const int32_t *key;
  int64_t key_step, n;
  uint32_t cut;
  double scale;
  // the strided form: extents, and the strides of x, residual and out
  int ndim;
  int64_t shape[DROP_MAXD], stride[3][DROP_MAXD];
};

template <class C>
__device__ __forceinline__ C drop_one(C x, bool keep, C scale) {
  return keep ? x * scale : 0;  // (chosen, not multiplied: a NaN that is dropped is gone)
}
// Which of the four elements of block `b` are kept.
struct Keep {
  bool k[4];
};
__device__ __forceinline__ Keep keep_four(uint32_t k0, uint32_t k1, uint64_t b, uint32_t cut) {
  uint32_t w0 = (uint32_t)b, w1 = (uint32_t)(b >> 32);
  threefry_block(k0, k1, w0, w1);
  return {{(w0 & 0xffffu) >= cut, (w0 >> 16) >= cut, (w1 & 0xffffu) >= cut, (w1 >> 16) >= cut}};
}

// All operands dense: a lane takes the elements of one or two blocks, 16 bytes of a 16- or 32-bit dtype.
template <int DT, bool RESIDUAL>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs a) {
  using IO = Io<DT>;
  using C = typename IO::C;
  using S = typename IO::S;
  constexpr int N = IO::V < 4 ? 4 : IO::V, L = N / IO::V;  // elements and vectors of a lane
  const uint32_t k0 = (uint32_t)a.key[0], k1 = (uint32_t)a.key[a.key_step];
  const C scale = (C)a.scale;
  const S *x = reinterpret_cast<const S *>(a.x), *r = reinterpret_cast<const S *>(a.residual);
  S *out = reinterpret_cast<S *>(a.out);
  for (int64_t first = ((int64_t)blockIdx.x * 256 + threadIdx.x) * N; first < a.n; first += (int64_t)gridDim.x * 256 * N) {
    if (first + N <= a.n) {
      Words xw[L], rw[L];
#pragma unroll
      for (int l = 0; l < L; l++) {
        xw[l] = load_words(x + first + l * IO::V);
        if (RESIDUAL) rw[l] = load_words(r + first + l * IO::V);
      }
      bool keep[N];
#pragma unroll
      for (int q = 0; q < N / 4; q++) {
        const Keep four = keep_four(k0, k1, (uint64_t)first / 4 + q, a.cut);
#pragma unroll
        for (int j = 0; j < 4; j++) keep[q * 4 + j] = four.k[j];
      }
#pragma unroll
      for (int l = 0; l < L; l++) {
        C y[IO::V], add[IO::V];
        IO::widen(xw[l], y);
        if (RESIDUAL) IO::widen(rw[l], add);
#pragma unroll
        for (int j = 0; j < IO::V; j++) {
          y[j] = drop_one(y[j], keep[l * IO::V + j], scale);
          if (RESIDUAL) y[j] = y[j] + add[j];
        }
        store_words(out + first + l * IO::V, IO::narrow(y));
      }
    } else {
      for (int64_t i = first; i < a.n; i++) {
        const Keep four = keep_four(k0, k1, (uint64_t)i / 4, a.cut);
        const int j = (int)(i & 3);
        C y = drop_one(IO::ld(x[i]), j < 2 ? (j ? four.k[1] : four.k[0]) : (j == 3 ? four.k[3] : four.k[2]), scale);
        if (RESIDUAL) y = y + IO::ld(r[i]);
        out[i] = IO::st(y);
      }
    }
  }
}

// Any strides: a lane takes one block. Its four elements lie in one row (the last dim) unless they
// cross its end; only then each has its own way through the extents.
template <int DT>
__global__ __launch_bounds__(256) void dropout_strided_kernel(DropoutArgs a) {
  using IO = Io<DT>;
  using C = typename IO::C;
  using S = typename IO::S;
  const S *x = reinterpret_cast<const S *>(a.x), *r = reinterpret_cast<const S *>(a.residual);
  S *out = reinterpret_cast<S *>(a.out);
  const bool small = a.n <= 0xffffffffLL;
  // the offsets of element i, and how many of its row are left from it on
  auto find = [&](int64_t i, int64_t (&at)[3]) -> int64_t {
    int64_t left = 1;
    at[0] = at[1] = at[2] = 0;
    for (int d = a.ndim - 1; d >= 0; d--) {
      const int64_t q = small ? (int64_t)((uint32_t)i / (uint32_t)a.shape[d]) : i / a.shape[d], at_d = i - q * a.shape[d];
      i = q;
      if (d == a.ndim - 1) left = a.shape[d] - at_d;
#pragma unroll
      for (int k = 0; k < 3; k++) at[k] += at_d * a.stride[k][d];
    }
    return left;
  };
  const uint32_t k0 = (uint32_t)a.key[0], k1 = (uint32_t)a.key[a.key_step];
  const C scale = (C)a.scale;
  const int last = a.ndim - 1;
  for (int64_t block = (int64_t)blockIdx.x * 256 + threadIdx.x; block * 4 < a.n; block += (int64_t)gridDim.x * 256) {
    const Keep keep = keep_four(k0, k1, (uint64_t)block, a.cut);
    int64_t at[3];
    const int64_t left = find(block * 4, at);
    if (left >= 4) {
      S xv[4], rv[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        xv[j] = x[at[0] + j * a.stride[0][last]];
        rv[j] = r ? r[at[1] + j * a.stride[1][last]] : S{};
      }
#pragma unroll
      for (int j = 0; j < 4; j++) {
        C y = drop_one(IO::ld(xv[j]), keep.k[j], scale);
        if (r) y = y + IO::ld(rv[j]);
        out[at[2] + j * a.stride[2][last]] = IO::st(y);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (block * 4 + j < a.n) {
          find(block * 4 + j, at);
          C y = drop_one(IO::ld(x[at[0]]), keep.k[j], scale);
          if (r) y = y + IO::ld(r[at[1]]);
          out[at[2]] = IO::st(y);
        }
    }
  }
}

// Drops extents of one and merges dims that compose on every operand.
void merge_dims(DropoutArgs &a) {
  int n = 0;
  for (int d = 0; d < a.ndim; d++) {
    if (a.shape[d] == 1) continue;
    bool composes = n > 0;
    for (int k = 0; k < 3 && composes; k++) composes = a.stride[k][n - 1] == a.stride[k][d] * a.shape[d];
    if (composes) a.shape[n - 1] *= a.shape[d];
    else a.shape[n++] = a.shape[d];
    for (int k = 0; k < 3; k++) a.stride[k][n - 1] = a.stride[k][d];
  }
  if (n == 0) {
    a.shape[0] = 1;
    for (int k = 0; k < 3; k++) a.stride[k][0] = 1;
    n = 1;
  }
  a.ndim = n;
}

template <int DT>
void launch(nxh_context *ctx, const DropoutArgs &a, bool dense) {
  constexpr int N = Io<DT>::V < 4 ? 4 : Io<DT>::V;
  const int64_t lanes = dense ? (a.n + N - 1) / N : (a.n + 3) / 4;
  const dim3 grid((unsigned)std::min<int64_t>((lanes + 255) / 256, DROP_BLOCKS));
  if (!dense) hipLaunchKernelGGL((dropout_strided_kernel<DT>), grid, dim3(256), 0, ctx->stream, a);
  else if (a.residual) hipLaunchKernelGGL((dropout_kernel<DT, true>), grid, dim3(256), 0, ctx->stream, a);
  else hipLaunchKernelGGL((dropout_kernel<DT, false>), grid, dim3(256), 0, ctx->stream, a);
}

}  // namespace

NXH_EXPORT int nxh_dropout(nxh_context *ctx, const nxh_tensor *out, const nxh_tensor *x, const nxh_tensor *residual,
                           const nxh_tensor *key, double rate) {
  NXH_DEFER_TOUCH(ctx, 1, out, x, residual, key);
  const char *op = "dropout";
  if (!ctx || !out || !x || !key) return nxh_fail(NXH_INVALID_ARGUMENT, op, "null argument");
  for (const nxh_tensor *t : {out, x, residual, key})
    if (t)
      if (int rc = nxh_check_tensor(op, t)) return rc;
  const int dt = x->dtype;
  if (!nxh_same_shape(out, x) || (residual && !nxh_same_shape(residual, x))) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
  if (key->ndim != 1 || key->shape[0] != 2) return nxh_fail(NXH_INVALID_ARGUMENT, op, "key must be two int32");
  if (!(rate >= 0.0 && rate <= 1.0)) return nxh_fail(NXH_INVALID_ARGUMENT, op, "rate must be between 0 and 1");
  if ((dt != NXH_F32 && dt != NXH_BF16 && dt != NXH_F16 && dt != NXH_F64) || out->dtype != dt ||
      (residual && residual->dtype != dt) || key->dtype != NXH_I32)
    return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
  for (int d = 0; d < out->ndim; d++)
    if (out->shape[d] > 1 && out->strides[d] == 0) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_OUT_ALIASED);
  DropoutArgs a;
  a.n = 1;
  a.ndim = x->ndim;
  for (int d = 0; d < x->ndim; d++)
    if (x->shape[d] == 0) return NXH_OK;
  for (int d = 0; d < x->ndim; d++) {
    a.shape[d] = x->shape[d];
    a.n *= x->shape[d];
    a.stride[0][d] = x->strides[d];
    a.stride[1][d] = residual ? residual->strides[d] : x->strides[d];
    a.stride[2][d] = out->strides[d];
  }
  merge_dims(a);
  const int64_t es = nxh_elem_size(dt);
  a.x = (const char *)x->data + x->offset * es;
  a.residual = residual ? (const char *)residual->data + residual->offset * es : nullptr;
  a.out = (char *)out->data + out->offset * es;
  a.key = (const int32_t *)key->data + key->offset;
  a.key_step = key->strides[0];
  a.cut = (uint32_t)std::floor(rate * 65536.0 + 0.5);
  a.scale = a.cut < 65536 ? 65536.0 / (65536.0 - a.cut) : 0.0;
  const bool dense = a.ndim == 1 && a.stride[0][0] == 1 && a.stride[1][0] == 1 && a.stride[2][0] == 1;
  std::lock_guard<std::mutex> guard(ctx->mu);
  NXH_HIP(op, hipSetDevice(ctx->device));
  nxh_set_path(dense ? "dropout" : "dropout_strided");
  if (dt == NXH_F32) launch<NXH_F32>(ctx, a, dense);
  else if (dt == NXH_BF16) launch<NXH_BF16>(ctx, a, dense);
  else if (dt == NXH_F16) launch<NXH_F16>(ctx, a, dense);
  else launch<NXH_F64>(ctx, a, dense);
  NXH_HIP(op, hipGetLastError());
  return NXH_OK;
}
