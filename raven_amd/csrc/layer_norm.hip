// layer_norm.hip — nxh_layer_norm: the layer norm that is differentiated, with the statistics
// that its gradient (layer_norm_grad.hip) takes:
//
//   mean = sum x / N,  rstd = 1 / sqrt(sum (x - mean)^2 / N + eps),  out = (x - mean) rstd gamma + beta
//
// Everything is held in float32 (float64 for float64) and rounded once, on the way out:
// nxh_layer_norm_rows is the other form, which rounds where the primitives do. The variance is that
// of the centred values, from registers: no difference of large sums.
//
// It reads x and writes out, once each: memory bounds it, at ten vector operations an element. [8192,768] bfloat16 6.2 us,
// [65536,768] 39.4 us (5.1 TB/s); of a few rows the launch is the time ([8,768]: 2.5 us on the device, 4.4 with the call).

#include <cmath>

#include "layer_norm_train.hpp"

namespace {

enum { LN_OUT, LN_X, LN_MEAN, LN_RSTD, LN_OPERANDS };
struct LayerNormArgs {
  RowGeom g;
  RowOperand o[LN_OPERANDS];  // mean, rstd: base may be null
  const char *gamma, *beta;   // null: ones, zeros
  double eps;
};

__device__ __forceinline__ float reciprocal_root(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double reciprocal_root(double v) { return 1.0 / sqrt(v); }

template <int DT, int G, int NV, Rows R>
__global__ __launch_bounds__(ln_threads(G)) void layer_norm_kernel(LayerNormArgs a) {
  using IO = Io<DT>;
  using C = typename IO::C;
  using S = typename IO::S;
  constexpr int V = IO::V, GROUPS = ln_threads(G) / G;
  __shared__ C lds[G > 64 ? G / 64 : 1];
  const int lane = threadIdx.x % G, n = a.g.n, nvec = (n + V - 1) / V;
  const S *gamma = reinterpret_cast<const S *>(a.gamma), *beta = reinterpret_cast<const S *>(a.beta);
  // Every lane loads for every v, a vector past the row as the row's last: a load under a condition is waited for before the next one.
  int c[NV];
#pragma unroll
  for (int v = 0; v < NV; v++) c[v] = v * G + lane < nvec ? v * G + lane : nvec - 1;
  Words gv[NV], bv[NV];
#pragma unroll
  for (int v = 0; v < NV; v++) {
    gv[v] = gamma ? load_part<R>(gamma, c[v], n) : IO::all(1);
    bv[v] = beta ? load_part<R>(beta, c[v], n) : IO::all(0);
  }
  // Whether this lane's vector v has element j for itself. Only the row's last vector may not: which v that is is the same for all lanes.
  const int last = (nvec - 1) / G;
  auto owns = [&](int v, int j) { return R == WHOLE || v != last || vec_owns<V, R>(c[v], j, n); };
  const C count = (C)n, eps = (C)a.eps;
  for (int64_t row = (int64_t)blockIdx.x * GROUPS + group_number<G, ln_threads(G)>(); row < a.g.rows; row += (int64_t)gridDim.x * GROUPS) {
    int64_t at[LN_OPERANDS];
    row_starts(a.g, (uint32_t)row, a.o, at);
    const S *x = reinterpret_cast<const S *>(a.o[LN_X].base) + at[LN_X];
    S *out = reinterpret_cast<S *>(const_cast<char *>(a.o[LN_OUT].base)) + at[LN_OUT];
    Words raw[NV];
#pragma unroll
    for (int v = 0; v < NV; v++) raw[v] = load_part<R>(x, c[v], n);
    C t[NV][V], s[1] = {0};
#pragma unroll
    for (int v = 0; v < NV; v++) {
      IO::widen(raw[v], t[v]);
      if (v * G + lane < nvec)
#pragma unroll
        for (int j = 0; j < V; j++) s[0] = s[0] + (owns(v, j) ? t[v][j] : 0);
    }
    group_combine<G>(s, Sum<C>{}, lds);
    const C mean = s[0] / count;
    s[0] = 0;
#pragma unroll
    for (int v = 0; v < NV; v++) {
#pragma unroll
      for (int j = 0; j < V; j++) t[v][j] = t[v][j] - mean;
      if (v * G + lane < nvec)
#pragma unroll
        for (int j = 0; j < V; j++) {
          const C own = owns(v, j) ? t[v][j] : 0;
          s[0] = fused(own, own, s[0]);
        }
    }
    group_combine<G>(s, Sum<C>{}, lds);
    const C rstd = reciprocal_root(s[0] / count + eps);
    if (lane == 0) {
      if (a.o[LN_MEAN].base) reinterpret_cast<C *>(const_cast<char *>(a.o[LN_MEAN].base))[at[LN_MEAN]] = mean;
      if (a.o[LN_RSTD].base) reinterpret_cast<C *>(const_cast<char *>(a.o[LN_RSTD].base))[at[LN_RSTD]] = rstd;
    }
#pragma unroll
    for (int v = 0; v < NV; v++) {
      C w[V], b[V];
      if constexpr (G * NV * V >= 1024 * 32) asm("" : "+v"(gv[v]), "+v"(bv[v]));  // (widened once for all rows they would take registers that there are not)
      IO::widen(gv[v], w);
      IO::widen(bv[v], b);
#pragma unroll
      for (int j = 0; j < V; j++) t[v][j] = fused(t[v][j] * rstd, w[j], b[j]);
      if (v * G + lane < nvec) store_part<R>(out, c[v], n, IO::narrow(t[v]));
    }
  }
}

// Rows that registers do not hold: a block walks its row three times, the second and the third time out of the caches.
constexpr int LONG_THREADS = 1024;
template <int DT>
__global__ __launch_bounds__(LONG_THREADS) void layer_norm_long_kernel(LayerNormArgs a) {
  using IO = Io<DT>;
  using C = typename IO::C;
  using S = typename IO::S;
  constexpr int V = IO::V;
  __shared__ C lds[LONG_THREADS / 64];
  const int n = a.g.n, nvec = (n + V - 1) / V;
  const S *gamma = reinterpret_cast<const S *>(a.gamma), *beta = reinterpret_cast<const S *>(a.beta);
  const C count = (C)n;
  for (int64_t row = blockIdx.x; row < a.g.rows; row += gridDim.x) {
    int64_t at[LN_OPERANDS];
    row_starts(a.g, (uint32_t)row, a.o, at);
    const S *x = reinterpret_cast<const S *>(a.o[LN_X].base) + at[LN_X];
    S *out = reinterpret_cast<S *>(const_cast<char *>(a.o[LN_OUT].base)) + at[LN_OUT];
    C s[1] = {0}, t[V];
    for (int c = threadIdx.x; c < nvec; c += LONG_THREADS) {
      IO::widen(load_part<RAGGED>(x, c, n), t);
#pragma unroll
      for (int j = 0; j < V; j++) s[0] = s[0] + (vec_owns<V, RAGGED>(c, j, n) ? t[j] : 0);
    }
    group_combine<LONG_THREADS>(s, Sum<C>{}, lds);
    const C mean = s[0] / count;
    s[0] = 0;
    for (int c = threadIdx.x; c < nvec; c += LONG_THREADS) {
      IO::widen(load_part<RAGGED>(x, c, n), t);
#pragma unroll
      for (int j = 0; j < V; j++) {
        const C own = vec_owns<V, RAGGED>(c, j, n) ? t[j] - mean : 0;
        s[0] = fused(own, own, s[0]);
      }
    }
    group_combine<LONG_THREADS>(s, Sum<C>{}, lds);
    const C rstd = reciprocal_root(s[0] / count + (C)a.eps);
    if (threadIdx.x == 0) {
      if (a.o[LN_MEAN].base) reinterpret_cast<C *>(const_cast<char *>(a.o[LN_MEAN].base))[at[LN_MEAN]] = mean;
      if (a.o[LN_RSTD].base) reinterpret_cast<C *>(const_cast<char *>(a.o[LN_RSTD].base))[at[LN_RSTD]] = rstd;
    }
    for (int c = threadIdx.x; c < nvec; c += LONG_THREADS) {
      C w[V], b[V];
      IO::widen(load_part<RAGGED>(x, c, n), t);
      IO::widen(gamma ? load_part<RAGGED>(gamma, c, n) : IO::all(1), w);
      IO::widen(beta ? load_part<RAGGED>(beta, c, n) : IO::all(0), b);
#pragma unroll
      for (int j = 0; j < V; j++) t[j] = fused((t[j] - mean) * rstd, w[j], b[j]);
      store_own(out, c, n, IO::narrow(t));
    }
  }
}

template <int DT, int G, int NV>
void launch(nxh_context *ctx, const LayerNormArgs &a) {
  constexpr int V = Io<DT>::V, GROUPS = ln_threads(G) / G;
  const int64_t most = (int64_t)(ctx->compute_units > 0 ? ctx->compute_units : 256) * (2048 / ln_threads(G));
  const dim3 grid((unsigned)std::min<int64_t>((a.g.rows + GROUPS - 1) / GROUPS, most));
  if (a.g.n % V == 0) hipLaunchKernelGGL((layer_norm_kernel<DT, G, NV, WHOLE>), grid, dim3(ln_threads(G)), 0, ctx->stream, a);
  else hipLaunchKernelGGL((layer_norm_kernel<DT, G, NV, G * NV == 1 ? SHORT : RAGGED>), grid, dim3(ln_threads(G)), 0, ctx->stream, a);
}
template <int DT>
void launch_rows(nxh_context *ctx, const LayerNormArgs &a) {
  constexpr int V = Io<DT>::V;
  const int nvec = (a.g.n + V - 1) / V;
#define X(G, NV) \
  if (nvec <= G * NV) return launch<DT, G, NV>(ctx, a);
  LN_GROUPS_FORWARD(X)
#undef X
  const dim3 grid((unsigned)std::min<int64_t>(a.g.rows, ctx->compute_units > 0 ? ctx->compute_units : 256));
  hipLaunchKernelGGL((layer_norm_long_kernel<DT>), grid, dim3(LONG_THREADS), 0, ctx->stream, a);
}

}  // namespace

NXH_EXPORT int nxh_layer_norm(nxh_context *ctx, const nxh_tensor *out, const nxh_tensor *mean, const nxh_tensor *rstd,
                              const nxh_tensor *x, const nxh_tensor *gamma, const nxh_tensor *beta, double eps) {
  NXH_DEFER_TOUCH(ctx, 3, out, mean, rstd, x, gamma, beta);
  const char *op = "layer_norm";
  if (!ctx || !out || !x) return nxh_fail(NXH_INVALID_ARGUMENT, op, "null argument");
  int rc = NXH_OK;
  for (const nxh_tensor *t : {out, mean, rstd, x, gamma, beta})
    if (t && (rc = nxh_check_tensor(op, t))) return rc;
  const int dx = x->dtype;
  LayerNormArgs a;
  if ((rc = same_shape(op, out, x)) || (rc = rows_geometry(op, x, a.g)) || (rc = out_rows_ok(op, out))) return rc;
  if (!(eps >= 0.0)) return nxh_fail(NXH_INVALID_ARGUMENT, op, "eps must be >= 0");
  if (!float_dtype_ok(dx) || out->dtype != dx || (gamma && gamma->dtype != dx) || (beta && beta->dtype != dx))
    return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
  for (const nxh_tensor *t : {mean, rstd})
    if (t && ((rc = row_values_ok(op, t, x, statistics_dtype(dx))) || (rc = out_rows_ok(op, t)))) return rc;
  for (const nxh_tensor *t : {gamma, beta})
    if (t && (rc = row_vector_ok(op, t, a.g.n))) return rc;
  // With as many rows as columns statistics have the shape of the weights, which blocks read at their start, while others already write.
  for (const nxh_tensor *t : {mean, rstd})
    for (const nxh_tensor *w : {gamma, beta})
      if (t && w && a.g.rows > 1 && same_view(t, w))
        return nxh_fail(NXH_INVALID_ARGUMENT, op, "mean and rstd must not replace gamma or beta");
  if (a.g.rows == 0) return NXH_OK;
  if (a.g.n == 0) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_EMPTY_REDUCE);
  if (!unit_stride(x) || !unit_stride(out)) return nxh_fail(NXH_FAILURE, op, "rows must be contiguous");
  row_operand(out, a.o[LN_OUT]);
  row_operand(x, a.o[LN_X]);
  row_value_operand(mean, a.o[LN_MEAN]);
  row_value_operand(rstd, a.o[LN_RSTD]);
  merge_outer_dims(a.g, {&a.o[LN_OUT], &a.o[LN_X], &a.o[LN_MEAN], &a.o[LN_RSTD]});
  const int64_t es = nxh_elem_size(dx);
  a.gamma = gamma ? (const char *)gamma->data + gamma->offset * es : nullptr;
  a.beta = beta ? (const char *)beta->data + beta->offset * es : nullptr;
  a.eps = eps;
  std::lock_guard<std::mutex> guard(ctx->mu);
  NXH_HIP(op, hipSetDevice(ctx->device));
  nxh_set_path(a.g.n > LN_VECTORS * (16 / es) ? "layer_norm_long" : "layer_norm");
  if (dx == NXH_F32) launch_rows<NXH_F32>(ctx, a);
  else if (dx == NXH_BF16) launch_rows<NXH_BF16>(ctx, a);
  else if (dx == NXH_F16) launch_rows<NXH_F16>(ctx, a);
  else launch_rows<NXH_F64>(ctx, a);
  NXH_HIP(op, hipGetLastError());
  return NXH_OK;
}
