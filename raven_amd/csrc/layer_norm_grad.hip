// layer_norm_grad.hip — nxh_layer_norm_grad: the transposed step of nxh_layer_norm. With
// h = (x - mean) rstd, w = g gamma and N the row's length:
//
//   dx = rstd (w - sum w / N - h sum (w h) / N),   dgamma = sum_rows g h,   dbeta = sum_rows g
//
// One pass over g and x makes all three. A group of lanes keeps a row in registers between its two
// sums and dx, and the sums over rows of the columns that its lanes hold from row to row; a block
// adds up its groups and writes one row of partial sums, a second launch adds those in a fixed order.
// Nothing is added by atomics, so equal calls give equal bits. All sums are float32 (float64 for float64).
//
// Memory bounds it: g and x in, dx out; the partial sums are held to some percent of that by the
// number of blocks. [65536,1024] bfloat16 79 us (5.1 TB/s), [16384,4096] 81 (5.0), [16384,16384] 311 (5.2). Of [8192,768], 11.5 us, a
// half does not go by the rows: 3.7 us from the launch to the end of a first row, 1.5 for the blocks' sums, 2.2 for the second launch.

#include "layer_norm_train.hpp"

namespace {

enum { LG_DX, LG_G, LG_X, LG_MEAN, LG_RSTD, LG_OPERANDS };
struct LayerNormGradArgs {
  RowGeom g;
  RowOperand o[LG_OPERANDS];  // dx: base may be null
  const char *gamma;          // null: ones
  void *partials;             // [blocks][2][n] sums of g h and of g; null: not wanted
};

// Adds up one value per lane over the groups of a wave: lanes with equal places in their groups.
template <int G, class C>
__device__ __forceinline__ C across_groups(C v) {
  const Sum<C> sum;
  if constexpr (G < 64) v = combine_step<32>(v, sum);
  if constexpr (G < 32) v = combine_step<16>(v, sum);
  if constexpr (G < 16) v = combine_step<8>(v, sum);
  if constexpr (G < 8) v = v + __shfl_xor(v, 4, 64);
  if constexpr (G < 4) v = combine_step<2>(v, sum);
  if constexpr (G < 2) v = combine_step<1>(v, sum);
  return v;
}

// A lane's sums of a vector of columns, as words. (Of a row's last vector those that it shares with the one before are made of the same
// elements in the same order there: equal bits.)
template <int DT>
__device__ __forceinline__ void store_sums(typename Tr<DT>::C *at, const typename Tr<DT>::C (&sums)[Io<DT>::V]) {
  using C = typename Tr<DT>::C;
  constexpr int E = VECTOR<C>;
#pragma unroll
  for (int k = 0; k < Io<DT>::V; k += E) {
    struct Plane { C s[E]; } p;
#pragma unroll
    for (int j = 0; j < E; j++) p.s[j] = sums[k + j];
    store_words(at + k, __builtin_bit_cast(Words, p));
  }
}

// Blocks of many waves where a row has a wave or less: the block's sums are one row of partial sums, whatever the number of its
// groups. Sixteen waves where a lane's 16 elements leave them the registers: those together keep the memory at work. Eight of them
// where it has more, each with its next row on the way while it finishes one. ([98304,64] float16 12.8 us with eight, 12.3 with
// sixteen; [65536,128] bfloat16 14.5 and 13.5; 24 elements of sixteen waves go to scratch memory: [8192,1536] bfloat16 18 and 54.)
// (float64 needs some three registers an element more.)
template <int DT, int G, int NV>
constexpr int lg_threads = G > 64 ? G : NV * Io<DT>::V * (DT == NXH_F64 ? 3 : 1) <= 16 ? 1024 : 512;

template <int DT, int G, int NV, Rows R>
__global__ __launch_bounds__((lg_threads<DT, G, NV>)) void layer_norm_grad_kernel(LayerNormGradArgs a) {
  using IO = Io<DT>;
  using C = typename IO::C;
  using S = typename IO::S;
  constexpr int V = IO::V, T = lg_threads<DT, G, NV>, GROUPS = T / G, W = T / 64;
  constexpr int HALF = 2 * W * G * V;
  __shared__ __align__(16) C lds[G > 64 ? 2 * (G / 64) : 2 * HALF];
  const int lane = threadIdx.x % G, n = a.g.n, nvec = (n + V - 1) / V;
  const S *gamma = reinterpret_cast<const S *>(a.gamma);
  // A lane of sixteen waves has 128 registers. Two vectors of a 16-bit dtype take 111 of them, four of float32 116, with one row at a time; one
  // vector takes 34 to 68 (float64 too) and would have room for the next row's, which has not been tried. Where a row is all sixteen waves'
  // gamma, which the caches have, is read with it.
  constexpr bool AHEAD = T < 1024, HELD = G < 1024;
  // Every lane loads for every v, a vector past the row as the row's last: a load under a condition is waited for before the next one.
  int c[NV];
  Words gain[NV], xr[NV], gr[NV];
  C dgamma[NV][V], dbeta[NV][V];
#pragma unroll
  for (int v = 0; v < NV; v++) {
    c[v] = v * G + lane < nvec ? v * G + lane : nvec - 1;
    if (HELD) gain[v] = gamma ? load_part<R>(gamma, c[v], n) : IO::all(1);
#pragma unroll
    for (int j = 0; j < V; j++) dgamma[v][j] = dbeta[v][j] = 0;
  }
  // Whether this lane's vector v has element j for itself. Only the row's last vector may not: which v that is is the same for all lanes.
  const int last = (nvec - 1) / G;
  auto owns = [&](int v, int j) { return R == WHOLE || v != last || vec_owns<V, R>(c[v], j, n); };
  const C count = (C)n;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  int64_t row = (int64_t)blockIdx.x * GROUPS + group_number<G, T>(), at[LG_OPERANDS];
  C mean = 0, rstd = 0;
  const S *x = nullptr, *g = nullptr;
  auto begin = [&](int64_t r) {
    row_starts(a.g, (uint32_t)r, a.o, at);
    x = reinterpret_cast<const S *>(a.o[LG_X].base) + at[LG_X];
    g = reinterpret_cast<const S *>(a.o[LG_G].base) + at[LG_G];
    mean = reinterpret_cast<const C *>(a.o[LG_MEAN].base)[at[LG_MEAN]];
    rstd = reinterpret_cast<const C *>(a.o[LG_RSTD].base)[at[LG_RSTD]];
  };
  auto request = [&](int v) {
    xr[v] = load_part<R>(x, c[v], n);
    gr[v] = load_part<R>(g, c[v], n);
    if (!HELD) gain[v] = gamma ? load_part<R>(gamma, c[v], n) : IO::all(1);
  };
  if (AHEAD && row < a.g.rows) {
    begin(row);
#pragma unroll
    for (int v = 0; v < NV; v++) request(v);
  }
  for (; row < a.g.rows; row += step) {
    if constexpr (!AHEAD) {
      begin(row);
#pragma unroll
      for (int v = 0; v < NV; v++) request(v);
    }
    const C mu = mean, rs = rstd;
    C h[NV][V], w[NV][V], s[2] = {0, 0};
#pragma unroll
    for (int v = 0; v < NV; v++) {
      C gv[V], gw[V];
      if constexpr (NV * V >= 32) asm("" : "+v"(gain[v]));  // (widened once for all rows it would take registers that there are not)
      IO::widen(xr[v], h[v]);
      IO::widen(gr[v], gv);
      IO::widen(gain[v], gw);
#pragma unroll
      for (int j = 0; j < V; j++) {
        h[v][j] = (h[v][j] - mu) * rs;
        w[v][j] = gv[j] * gw[j];
        dgamma[v][j] = fused(gv[j], h[v][j], dgamma[v][j]);  // (of a lane with no vector v: never looked at)
        dbeta[v][j] = dbeta[v][j] + gv[j];
      }
      if (v * G + lane < nvec)
#pragma unroll
        for (int j = 0; j < V; j++) {
          const bool own = owns(v, j);
          s[0] = s[0] + (own ? w[v][j] : 0);
          s[1] = fused(own ? w[v][j] : 0, own ? h[v][j] : 0, s[1]);
        }
    }
    S *dx = reinterpret_cast<S *>(const_cast<char *>(a.o[LG_DX].base)) + at[LG_DX];
    if constexpr (AHEAD) {
      begin(row + step < a.g.rows ? row + step : row);  // (behind the last row its own again, for nothing)
#pragma unroll
      for (int v = 0; v < NV; v++) request(v);  // in flight while this row is finished
    }
    group_combine<G>(s, Sum<C>{}, lds);
    if (a.o[LG_DX].base) {
      const C c1 = s[0] / count, c2 = s[1] / count;
#pragma unroll
      for (int v = 0; v < NV; v++) {
#pragma unroll
        for (int j = 0; j < V; j++) w[v][j] = rs * fused(-h[v][j], c2, w[v][j] - c1);
        if (v * G + lane < nvec) store_part<R>(dx, c[v], n, IO::narrow(w[v]));
      }
    }
  }
  if (!a.partials) return;
  C *mine = reinterpret_cast<C *>(a.partials) + (int64_t)blockIdx.x * 2 * n;
  if constexpr (G > 64) {  // the block's only group
#pragma unroll
    for (int v = 0; v < NV; v++)
      if (v * G + lane < nvec) {
        store_sums<DT>(mine + vec_start<V, R>(c[v], n), dgamma[v]);
        store_sums<DT>(mine + n + vec_start<V, R>(c[v], n), dbeta[v]);
      }
  } else {
    // A wave's sums lie in planes of 16 bytes a lane: [wave][dgamma, dbeta][plane][lane][element of the plane].
    constexpr int E = 16 / (int)sizeof(C), P = (V + E - 1) / E, WAVE = 2 * P * G * E;
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int first = 0; first < NV; first += 2) {  // two vectors a barrier, as there is room
      if (first > 0) __syncthreads();
#pragma unroll
      for (int v = first; v < NV && v < first + 2; v++)
#pragma unroll
        for (int q = 0; q < P; q++) {
          struct alignas(16) Plane { C s[E]; } p, r;
#pragma unroll
          for (int j = 0; j < E; j++) {
            p.s[j] = across_groups<G>(dgamma[v][q * E + j]);
            r.s[j] = across_groups<G>(dbeta[v][q * E + j]);
          }
          if ((threadIdx.x & 63) < G) {
            C *at = lds + (v - first) * HALF + wave * WAVE + (q * G + lane) * E;
            *reinterpret_cast<Plane *>(at) = p;
            *reinterpret_cast<Plane *>(at + P * G * E) = r;
          }
        }
      __syncthreads();
#pragma unroll
      for (int v = first; v < NV && v < first + 2; v++)
        for (int e = threadIdx.x; e < WAVE; e += T) {
          const C *at = lds + (v - first) * HALF + e;
          C s = at[0];
#pragma unroll
          for (int k = 1; k < W; k++) s = s + at[k * WAVE];
          const int which = e / (P * G * E), i = v * G + e / E % G, j = e / (G * E) % P * E + e % E;
          if (i < nvec && vec_owns<V, R>(i, j, n)) mine[which * n + vec_start<V, R>(i, n) + j] = s;
        }
    }
  }
}

// ── rows that registers do not hold ─────────────────────────────────────────
// The rows' sums and dx by a block per row, which walks it twice; the columns' sums by blocks of 256 lanes that
// own a vector of columns each and walk a share of the rows: g and x are read again, which such rows have caches for.
constexpr int LONG_THREADS = 1024;
template <int DT>
__global__ __launch_bounds__(LONG_THREADS) void layer_norm_grad_long_kernel(LayerNormGradArgs a) {
  using IO = Io<DT>;
  using C = typename IO::C;
  using S = typename IO::S;
  constexpr int V = IO::V;
  __shared__ C lds[2 * (LONG_THREADS / 64)];
  const int n = a.g.n, nvec = (n + V - 1) / V;
  const S *gamma = reinterpret_cast<const S *>(a.gamma);
  const C count = (C)n;
  for (int64_t row = blockIdx.x; row < a.g.rows; row += gridDim.x) {
    int64_t at[LG_OPERANDS];
    row_starts(a.g, (uint32_t)row, a.o, at);
    const S *x = reinterpret_cast<const S *>(a.o[LG_X].base) + at[LG_X];
    const S *g = reinterpret_cast<const S *>(a.o[LG_G].base) + at[LG_G];
    S *dx = reinterpret_cast<S *>(const_cast<char *>(a.o[LG_DX].base)) + at[LG_DX];
    const C mu = reinterpret_cast<const C *>(a.o[LG_MEAN].base)[at[LG_MEAN]];
    const C rs = reinterpret_cast<const C *>(a.o[LG_RSTD].base)[at[LG_RSTD]];
    C s[2] = {0, 0};
    auto walk = [&](auto &&body) {
      for (int c = threadIdx.x; c < nvec; c += LONG_THREADS) {
        C h[V], w[V], gain[V];
        IO::widen(load_part<RAGGED>(x, c, n), h);
        IO::widen(load_part<RAGGED>(g, c, n), w);
        IO::widen(gamma ? load_part<RAGGED>(gamma, c, n) : IO::all(1), gain);
#pragma unroll
        for (int j = 0; j < V; j++) {
          h[j] = (h[j] - mu) * rs;
          w[j] = w[j] * gain[j];
        }
        body(c, h, w);
      }
    };
    walk([&](int c, const C *h, const C *w) {
#pragma unroll
      for (int j = 0; j < V; j++) {
        const bool own = vec_owns<V, RAGGED>(c, j, n);
        s[0] = s[0] + (own ? w[j] : 0);
        s[1] = fused(own ? w[j] : 0, own ? h[j] : 0, s[1]);
      }
    });
    group_combine<LONG_THREADS>(s, Sum<C>{}, lds);
    const C c1 = s[0] / count, c2 = s[1] / count;
    walk([&](int c, const C *h, const C *w) {
      C d[V];
#pragma unroll
      for (int j = 0; j < V; j++) d[j] = rs * fused(-h[j], c2, w[j] - c1);
      store_own(dx, c, n, IO::narrow(d));
    });
  }
}
template <int DT>
__global__ __launch_bounds__(256) void layer_norm_columns_kernel(LayerNormGradArgs a, int64_t share) {
  using IO = Io<DT>;
  using C = typename IO::C;
  using S = typename IO::S;
  constexpr int V = IO::V;
  const int n = a.g.n, c = blockIdx.x * 256 + threadIdx.x;
  if ((int64_t)c * V >= n) return;
  C dgamma[V], dbeta[V];
#pragma unroll
  for (int j = 0; j < V; j++) dgamma[j] = dbeta[j] = 0;
  const int64_t first = (int64_t)blockIdx.y * share, end = first + share < a.g.rows ? first + share : a.g.rows;
#pragma unroll 4
  for (int64_t row = first; row < end; row++) {
    int64_t at[LG_OPERANDS];
    row_starts(a.g, (uint32_t)row, a.o, at);
    C x[V], g[V];
    IO::widen(load_part<RAGGED>(reinterpret_cast<const S *>(a.o[LG_X].base) + at[LG_X], c, n), x);
    IO::widen(load_part<RAGGED>(reinterpret_cast<const S *>(a.o[LG_G].base) + at[LG_G], c, n), g);
    const C mu = reinterpret_cast<const C *>(a.o[LG_MEAN].base)[at[LG_MEAN]];
    const C rs = reinterpret_cast<const C *>(a.o[LG_RSTD].base)[at[LG_RSTD]];
#pragma unroll
    for (int j = 0; j < V; j++) {
      dgamma[j] = fused(g[j], (x[j] - mu) * rs, dgamma[j]);
      dbeta[j] = dbeta[j] + g[j];
    }
  }
  C *mine = reinterpret_cast<C *>(a.partials) + (int64_t)blockIdx.y * 2 * n + vec_start<V, RAGGED>(c, n);
  store_sums<DT>(mine, dgamma);
  store_sums<DT>(mine + n, dbeta);
}

// ── the partial sums ────────────────────────────────────────────────────────
// 32 columns of a block: a lane adds a vector of them from every 128th partial sum (every 64th of float64), and the lanes' sums are
// added in order.
struct JoinArgs {
  const void *partials;
  int64_t blocks;
  int n;
  char *out[2];  // dgamma, dbeta; null: not wanted
  int64_t stride[2];
};
template <int DT>
__global__ __launch_bounds__(1024) void layer_norm_join_kernel(JoinArgs a) {
  using IO = Io<DT>;
  using C = typename IO::C;
  using S = typename IO::S;
  constexpr int V = VECTOR<C>, LANES = 32 / V, PARTS = 1024 / LANES, W = 16;
  __shared__ C lds[W][32];
  const int lane = threadIdx.x % LANES, part = threadIdx.x / LANES;
  const int64_t columns = 2 * (int64_t)a.n, first = (int64_t)blockIdx.x * 32 + lane * V;
  const C *p = reinterpret_cast<const C *>(a.partials);
  C s[V];
#pragma unroll
  for (int j = 0; j < V; j++) s[j] = 0;
  if (first + V <= columns) {
#pragma unroll 4
    for (int64_t b = part; b < a.blocks; b += PARTS) {
      struct Elements { C x[V]; } e = __builtin_bit_cast(Elements, load_words(p + b * columns + first));
#pragma unroll
      for (int j = 0; j < V; j++) s[j] = s[j] + e.x[j];
    }
  } else {
    for (int64_t b = part; b < a.blocks; b += PARTS)
#pragma unroll
      for (int j = 0; j < V; j++)
        if (first + j < columns) s[j] = s[j] + p[b * columns + first + j];
  }
#pragma unroll
  for (int j = 0; j < V; j++) {
    s[j] = across_groups<LANES>(s[j]);
    if ((threadIdx.x & 63) < LANES) lds[threadIdx.x >> 6][lane * V + j] = s[j];
  }
  __syncthreads();
  const int64_t column = (int64_t)blockIdx.x * 32 + threadIdx.x;
  if (threadIdx.x >= 32 || column >= columns) return;
  C sum = lds[0][threadIdx.x];
#pragma unroll
  for (int w = 1; w < W; w++) sum = sum + lds[w][threadIdx.x];
  const int which = column >= a.n;
  char *out = which ? a.out[1] : a.out[0];
  const int64_t stride = which ? a.stride[1] : a.stride[0];
  if (out) reinterpret_cast<S *>(out)[(column - (which ? a.n : 0)) * stride] = IO::st(sum);
}

// ── host side ───────────────────────────────────────────────────────────────
struct Plan {
  void (*launch)(nxh_context *, const LayerNormGradArgs &, int64_t blocks);
  int64_t blocks;  // rows of partial sums
};
template <int DT, int G, int NV>
void launch(nxh_context *ctx, const LayerNormGradArgs &a, int64_t blocks) {
  constexpr int V = Io<DT>::V;
  const dim3 grid((unsigned)blocks);
  if (a.g.n % V == 0) hipLaunchKernelGGL((layer_norm_grad_kernel<DT, G, NV, WHOLE>), grid, dim3((lg_threads<DT, G, NV>)), 0, ctx->stream, a);
  else hipLaunchKernelGGL((layer_norm_grad_kernel<DT, G, NV, G * NV == 1 ? SHORT : RAGGED>), grid, dim3((lg_threads<DT, G, NV>)), 0, ctx->stream, a);
}
template <int DT>
void launch_long(nxh_context *ctx, const LayerNormGradArgs &a, int64_t blocks) {
  constexpr int V = Io<DT>::V;
  const int64_t units = ctx->compute_units > 0 ? ctx->compute_units : 256;
  if (a.partials) {  // before dx, which may go where g or x is
    const dim3 grid((unsigned)(((a.g.n + V - 1) / V + 255) / 256), (unsigned)blocks);
    hipLaunchKernelGGL((layer_norm_columns_kernel<DT>), grid, dim3(256), 0, ctx->stream, a, (a.g.rows + blocks - 1) / blocks);
  }
  if (a.o[LG_DX].base)
    hipLaunchKernelGGL((layer_norm_grad_long_kernel<DT>), dim3((unsigned)std::min(a.g.rows, units)), dim3(LONG_THREADS), 0, ctx->stream, a);
}
// A block for each unit: another one has partial sums of its own, which are to be written and read. It pays where blocks of four waves keep
// too little on its way, with many rows ([30000,3600] bfloat16 157 us with one, 127 with two; [16384,8192], twice the vectors a lane, 161 and
// 164; [1024,4096] 15 and 19).
template <int DT>
Plan plan(nxh_context *ctx, int n, int64_t rows) {
  constexpr int V = Io<DT>::V;
  const int64_t units = ctx->compute_units > 0 ? ctx->compute_units : 256;
  const int nvec = (n + V - 1) / V;
#define X(G, NV)                                                                                                \
  if (nvec <= G * NV)                                                                                           \
    return {launch<DT, G, NV>, std::min((rows + lg_threads<DT, G, NV> / G - 1) / (lg_threads<DT, G, NV> / G), units * (G == 256 && NV == 2 && rows > 16 * units ? 2 : 1))};
  LN_GROUPS_GRAD(X)
  if constexpr (V < 8) {
    LN_GROUPS_GRAD_WORDS(X)
  }
#undef X
  const int64_t tiles = (nvec + 255) / 256;
  return {launch_long<DT>, std::max<int64_t>(1, std::min(rows / 8, 2 * units / tiles))};
}

}  // namespace

NXH_EXPORT int nxh_layer_norm_grad(nxh_context *ctx, const nxh_tensor *dx, const nxh_tensor *dgamma, const nxh_tensor *dbeta,
                                   const nxh_tensor *g, const nxh_tensor *x, const nxh_tensor *mean, const nxh_tensor *rstd,
                                   const nxh_tensor *gamma) {
  NXH_DEFER_TOUCH(ctx, 3, dx, dgamma, dbeta, g, x, mean, rstd, gamma);
  const char *op = "layer_norm_grad";
  if (!ctx || !g || !x || !mean || !rstd || (!dx && !dgamma && !dbeta)) return nxh_fail(NXH_INVALID_ARGUMENT, op, "null argument");
  int rc = NXH_OK;
  for (const nxh_tensor *t : {dx, dgamma, dbeta, g, x, mean, rstd, gamma})
    if (t && (rc = nxh_check_tensor(op, t))) return rc;
  const int dt = x->dtype;
  LayerNormGradArgs a;
  if ((rc = same_shape(op, g, x)) || (dx && (rc = same_shape(op, dx, x))) || (rc = rows_geometry(op, x, a.g))) return rc;
  for (const nxh_tensor *t : {dx, dgamma, dbeta})
    if (t && (rc = out_rows_ok(op, t))) return rc;
  if (!float_dtype_ok(dt)) return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
  for (const nxh_tensor *t : {dx, dgamma, dbeta, g, gamma})
    if (t && t->dtype != dt) return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
  for (const nxh_tensor *t : {mean, rstd})
    if ((rc = row_values_ok(op, t, x, statistics_dtype(dt)))) return rc;
  if (gamma && (rc = row_vector_ok(op, gamma, a.g.n))) return rc;
  for (const nxh_tensor *t : {dgamma, dbeta})
    if (t && (t->ndim != 1 || t->shape[0] != a.g.n)) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
  if (a.g.rows > 0 && a.g.n == 0) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_EMPTY_REDUCE);
  if (a.g.n == 0) return NXH_OK;
  if (a.g.rows > 0 && (!unit_stride(x) || !unit_stride(g) || (dx && !unit_stride(dx))))
    return nxh_fail(NXH_FAILURE, op, "rows must be contiguous");
  row_operand(dx, a.o[LG_DX]);
  row_operand(g, a.o[LG_G]);
  row_operand(x, a.o[LG_X]);
  row_value_operand(mean, a.o[LG_MEAN]);
  row_value_operand(rstd, a.o[LG_RSTD]);
  merge_outer_dims(a.g, {&a.o[LG_DX], &a.o[LG_G], &a.o[LG_X], &a.o[LG_MEAN], &a.o[LG_RSTD]});
  const int64_t es = nxh_elem_size(dt);
  a.gamma = gamma ? (const char *)gamma->data + gamma->offset * es : nullptr;
  a.partials = nullptr;
  std::lock_guard<std::mutex> guard(ctx->mu);
  NXH_HIP(op, hipSetDevice(ctx->device));
  const bool weights = dgamma || dbeta;
  nxh_set_path(a.g.n > ln_vectors_grad((int)es) * (16 / es) ? "layer_norm_grad_long" : "layer_norm_grad");
  Plan p{nullptr, 0};  // no rows: sums of nothing
  if (a.g.rows > 0)
    p = dt == NXH_F32 ? plan<NXH_F32>(ctx, a.g.n, a.g.rows) : dt == NXH_BF16 ? plan<NXH_BF16>(ctx, a.g.n, a.g.rows)
        : dt == NXH_F16 ? plan<NXH_F16>(ctx, a.g.n, a.g.rows) : plan<NXH_F64>(ctx, a.g.n, a.g.rows);
  if (weights && p.launch)
    if ((rc = nxh_alloc_locked(ctx, (size_t)p.blocks * 2 * (size_t)a.g.n * (dt == NXH_F64 ? 8 : 4), &a.partials))) return rc;
  if (p.launch) p.launch(ctx, a, p.blocks);
  if (weights) {
    JoinArgs j{a.partials, p.blocks, a.g.n, {nullptr, nullptr}, {1, 1}};
    const nxh_tensor *outs[2] = {dgamma, dbeta};
    for (int k = 0; k < 2; k++)
      if (outs[k]) {
        j.out[k] = (char *)outs[k]->data + outs[k]->offset * es;
        j.stride[k] = outs[k]->strides[0];
      }
    const dim3 grid((unsigned)((2 * (int64_t)a.g.n + 31) / 32));
    if (dt == NXH_F32) hipLaunchKernelGGL((layer_norm_join_kernel<NXH_F32>), grid, dim3(1024), 0, ctx->stream, j);
    else if (dt == NXH_BF16) hipLaunchKernelGGL((layer_norm_join_kernel<NXH_BF16>), grid, dim3(1024), 0, ctx->stream, j);
    else if (dt == NXH_F16) hipLaunchKernelGGL((layer_norm_join_kernel<NXH_F16>), grid, dim3(1024), 0, ctx->stream, j);
    else hipLaunchKernelGGL((layer_norm_join_kernel<NXH_F64>), grid, dim3(1024), 0, ctx->stream, j);
    if (a.partials) nxh_free_locked(ctx, a.partials);  // (the stream orders its next use behind these launches)
  }
  NXH_HIP(op, hipGetLastError());
  return NXH_OK;
}
