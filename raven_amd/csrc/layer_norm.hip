// layer_norm.hip — nxh_layer_norm: the layer norm that is differentiated, with the statistics
// that its gradient (layer_norm_grad.hip) takes:
//
//   mean = sum x / N,  rstd = 1 / sqrt(sum (x - mean)^2 / N + eps),  out = (x - mean) rstd gamma + beta
//
// Everything is held in float32 (float64 for float64) and rounded once, on the way out:
// nxh_layer_norm_rows is the other form, which rounds where the primitives do. The variance is that
// of the centred values, from registers: no difference of large sums.
//
// It reads x and writes out, once each: memory bounds it, at ten vector operations an element.

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

template <int DT, int G, int NV, bool RAGGED>
__global__ __launch_bounds__(ln_threads(G)) void layer_norm_kernel(LayerNormArgs a) {
  using TX = Tr<DT>;
  using C = typename TX::C;
  using S = typename TX::S;
  constexpr int V = VECTOR<S>, GROUPS = ln_threads(G) / G;
  __shared__ C lds[G > 64 ? G / 64 : 1];
  const int lane = threadIdx.x % G, n = a.g.n, nvec = (n + V - 1) / V;
  const S *gamma = reinterpret_cast<const S *>(a.gamma), *beta = reinterpret_cast<const S *>(a.beta);
  Vec<S, V> gv[NV], bv[NV];
#pragma unroll
  for (int v = 0; v < NV; v++) {
    const int c = v * G + lane;
    if (c < nvec && gamma) gv[v] = load_part<V, RAGGED>(gamma, c, n, S{});
    if (c < nvec && beta) bv[v] = load_part<V, RAGGED>(beta, c, n, S{});
  }
  const C count = (C)n, eps = (C)a.eps;
  for (int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / G; row < a.g.rows; row += (int64_t)gridDim.x * GROUPS) {
    int64_t at[LN_OPERANDS];
    row_starts(a.g, (uint32_t)row, a.o, at);
    const S *x = reinterpret_cast<const S *>(a.o[LN_X].base) + at[LN_X];
    S *out = reinterpret_cast<S *>(const_cast<char *>(a.o[LN_OUT].base)) + at[LN_OUT];
    Vec<S, V> raw[NV];
#pragma unroll
    for (int v = 0; v < NV; v++)
      if (v * G + lane < nvec) raw[v] = load_part<V, RAGGED>(x, v * G + lane, n, S{});
    C t[NV][V], s[1] = {0};
#pragma unroll
    for (int v = 0; v < NV; v++)
      if (v * G + lane < nvec)
#pragma unroll
        for (int j = 0; j < V; j++) {
          t[v][j] = TX::ld(raw[v].v[j]);
          s[0] = s[0] + t[v][j];  // (what is past the row's end was read as zero)
        }
    group_combine<G>(s, Sum<C>{}, lds);
    const C mean = s[0] / count;
    s[0] = 0;
#pragma unroll
    for (int v = 0; v < NV; v++)
      if (v * G + lane < nvec)
#pragma unroll
        for (int j = 0; j < V; j++) {
          t[v][j] = t[v][j] - mean;
          if (RAGGED && (v * G + lane) * V + j >= n) t[v][j] = 0;
          s[0] = fused(t[v][j], t[v][j], s[0]);
        }
    group_combine<G>(s, Sum<C>{}, lds);
    const C rstd = reciprocal_root(s[0] / count + eps);
    if (lane == 0) {
      if (a.o[LN_MEAN].base) reinterpret_cast<C *>(const_cast<char *>(a.o[LN_MEAN].base))[at[LN_MEAN]] = mean;
      if (a.o[LN_RSTD].base) reinterpret_cast<C *>(const_cast<char *>(a.o[LN_RSTD].base))[at[LN_RSTD]] = rstd;
    }
#pragma unroll
    for (int v = 0; v < NV; v++)
      if (v * G + lane < nvec) {
        Vec<S, V> o;
#pragma unroll
        for (int j = 0; j < V; j++) {
          C y = t[v][j] * rstd;
          if (gamma && beta) y = fused(y, TX::ld(gv[v].v[j]), TX::ld(bv[v].v[j]));
          else if (gamma) y = y * TX::ld(gv[v].v[j]);
          else if (beta) y = y + TX::ld(bv[v].v[j]);
          o.v[j] = TX::st(y);
        }
        store_part<V, RAGGED>(out, v * G + lane, n, o);
      }
  }
}

// Rows that registers do not hold: a block walks its row three times, the second and the third time out of the caches.
constexpr int LONG_THREADS = 1024;
template <int DT>
__global__ __launch_bounds__(LONG_THREADS) void layer_norm_long_kernel(LayerNormArgs a) {
  using TX = Tr<DT>;
  using C = typename TX::C;
  using S = typename TX::S;
  constexpr int V = VECTOR<S>;
  __shared__ C lds[LONG_THREADS / 64];
  const int n = a.g.n, nvec = (n + V - 1) / V;
  const S *gamma = reinterpret_cast<const S *>(a.gamma), *beta = reinterpret_cast<const S *>(a.beta);
  const C count = (C)n;
  for (int64_t row = blockIdx.x; row < a.g.rows; row += gridDim.x) {
    int64_t at[LN_OPERANDS];
    row_starts(a.g, (uint32_t)row, a.o, at);
    const S *x = reinterpret_cast<const S *>(a.o[LN_X].base) + at[LN_X];
    S *out = reinterpret_cast<S *>(const_cast<char *>(a.o[LN_OUT].base)) + at[LN_OUT];
    C s[1] = {0};
    for (int c = threadIdx.x; c < nvec; c += LONG_THREADS) {
      const Vec<S, V> raw = load_part<V, true>(x, c, n, S{});
#pragma unroll
      for (int j = 0; j < V; j++) s[0] = s[0] + TX::ld(raw.v[j]);
    }
    group_combine<LONG_THREADS>(s, Sum<C>{}, lds);
    const C mean = s[0] / count;
    s[0] = 0;
    for (int c = threadIdx.x; c < nvec; c += LONG_THREADS) {
      const Vec<S, V> raw = load_part<V, true>(x, c, n, S{});
#pragma unroll
      for (int j = 0; j < V; j++) {
        const C t = c * V + j < n ? TX::ld(raw.v[j]) - mean : 0;
        s[0] = fused(t, t, s[0]);
      }
    }
    group_combine<LONG_THREADS>(s, Sum<C>{}, lds);
    const C rstd = reciprocal_root(s[0] / count + (C)a.eps);
    if (threadIdx.x == 0) {
      if (a.o[LN_MEAN].base) reinterpret_cast<C *>(const_cast<char *>(a.o[LN_MEAN].base))[at[LN_MEAN]] = mean;
      if (a.o[LN_RSTD].base) reinterpret_cast<C *>(const_cast<char *>(a.o[LN_RSTD].base))[at[LN_RSTD]] = rstd;
    }
    for (int c = threadIdx.x; c < nvec; c += LONG_THREADS) {
      const Vec<S, V> raw = load_part<V, true>(x, c, n, S{});
      Vec<S, V> gv, bv, o;
      if (gamma) gv = load_part<V, true>(gamma, c, n, S{});
      if (beta) bv = load_part<V, true>(beta, c, n, S{});
#pragma unroll
      for (int j = 0; j < V; j++) {
        C y = (TX::ld(raw.v[j]) - mean) * rstd;
        if (gamma && beta) y = fused(y, TX::ld(gv.v[j]), TX::ld(bv.v[j]));
        else if (gamma) y = y * TX::ld(gv.v[j]);
        else if (beta) y = y + TX::ld(bv.v[j]);
        o.v[j] = TX::st(y);
      }
      store_part<V, true>(out, c, n, o);
    }
  }
}

template <int DT, int G, int NV>
void launch(nxh_context *ctx, const LayerNormArgs &a) {
  constexpr int V = VECTOR<typename Tr<DT>::S>, GROUPS = ln_threads(G) / G;
  const int64_t most = (int64_t)(ctx->compute_units > 0 ? ctx->compute_units : 256) * (2048 / ln_threads(G));
  const dim3 grid((unsigned)std::min<int64_t>((a.g.rows + GROUPS - 1) / GROUPS, most));
  if (a.g.n % V == 0) hipLaunchKernelGGL((layer_norm_kernel<DT, G, NV, false>), grid, dim3(ln_threads(G)), 0, ctx->stream, a);
  else hipLaunchKernelGGL((layer_norm_kernel<DT, G, NV, true>), grid, dim3(ln_threads(G)), 0, ctx->stream, a);
}
template <int DT>
void launch_rows(nxh_context *ctx, const LayerNormArgs &a) {
  constexpr int V = VECTOR<typename Tr<DT>::S>;
  const int nvec = (a.g.n + V - 1) / V;
#define X(G, NV) \
  if (nvec <= G * NV) return launch<DT, G, NV>(ctx, a);
  LN_GROUPS(X)
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
