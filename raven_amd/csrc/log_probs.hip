// log_probs.hip — the loss over a vocabulary: nxh_log_probs, nxh_log_probs_grad and
// nxh_log_probs_with_grad. For a row x of logits, with peak = max x and total = sum e^(x - peak):
//
//   log_p   = x[token] - peak - log total
//   entropy = log total - sum e^(x - peak) (x - peak) / total
//   d x     = g (1[token] - p) - g_entropy p (log p + entropy),  p = e^(x - peak) / total
//
// and the k largest x, equal ones by index. Nothing of the size of the logits is written but d x.
//
// One walk over the row keeps, lane by lane, the largest element so far and the two sums against it,
// rescaled where a vector of 16 bytes brings a larger one; the lanes' triples are then joined. Both sums
// have terms of one sign, so nothing cancels, and peak and total are given out apart: x - peak is exact
// near the peak, where x - log(sum e^x) would round to the step of the logarithm. Memory bounds it: the
// logits once; the gradient once more in and out. Five alternatives of [2048,50257] float32 75 us (5.5 TB/s);
// [8192,50257] bfloat16 statistics 152 to 159 us (5.2 to 5.4 TB/s, on three inputs in turn; 141 on one), both at once 318
// (5.2), the gradient by itself 290 (5.7).
//
// Exponentials are powers of two: with L = log2 e and the reference A = peak L as it rounds, 2^(x L - A) is one
// fused step and one instruction. What A lost in rounding, r = peak L - A, is a factor 2^r of every term: the
// sums are freed of it at the end, a quotient of two terms never has it.

#include <type_traits>
#include <utility>

#include "lane_groups.hpp"
#include "rows.hpp"

namespace {

enum { LP_X, LP_TOKEN, LP_LOG_P, LP_ENTROPY, LP_PEAK, LP_TOTAL, LP_TOP_LOG_P, LP_TOP_TOKEN, LP_G, LP_G_ENTROPY, LP_D, LP_OPERANDS };
struct LogProbsArgs {
  RowGeom g;
  RowOperand o[LP_OPERANDS];  // null where an operand is not there
  int top;
};
// Where the row begins in every operand.
struct Places {
  int64_t at[LP_OPERANDS];
};
template <class T>
__device__ __forceinline__ T *place(const LogProbsArgs &a, const Places &p, int k) {
  return reinterpret_cast<T *>(const_cast<char *>(a.o[k].base)) + p.at[k];
}

template <class C> struct Bounds;
// wide: rows whose largest element is no further from zero have an r below 1 and sums that cannot overflow; others are walked by
// differences (of finite values near the dtype's ends, or with infinities). low: the least reference, which a lane of
// lesser elements takes: beside a row's largest they count for nothing. none: 2^none is 0.
template <> struct Bounds<float> {
  static constexpr float wide = 0x1p20f, low = -0x1p21f, none = -300.0f, inf = __builtin_inff(), L = 0x1.715476p+0f, ln2 = 0x1.62e43p-1f;
};
template <> struct Bounds<double> {
  static constexpr double wide = 0x1p20, low = -0x1p21, none = -2000.0, inf = __builtin_inf(), L = 0x1.71547652b82fep+0, ln2 = 0x1.62e42fefa39efp-1;
};
__device__ __forceinline__ float power(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ double power(double x) { return exp2(x); }
__device__ __forceinline__ float larger(float a, float b) { return __builtin_fmaxf(a, b); }  // (a NaN is passed over: the sums have it)
__device__ __forceinline__ double larger(double a, double b) { return __builtin_fmax(a, b); }
template <class C>
struct Larger {
  __device__ __forceinline__ C operator()(C a, C b) const { return larger(a, b); }
};
template <class C>
__device__ __forceinline__ C reference(C peak) { return larger(peak * Bounds<C>::L, Bounds<C>::low); }
// Whether a row with this largest element is walked by its reference.
template <class C>
__device__ __forceinline__ bool is_near(C peak) { return __builtin_fabs(peak) <= Bounds<C>::wide; }

// How a row of n elements is cut: vectors that lie on 16 bytes, and single elements in front of the first and behind the last of them
// (of [8192,50257] contiguous bfloat16 logits seven rows in eight begin off 16 bytes: 173 us by vectors from their first
// element on, 141 by vectors that lie on 16 bytes). A group of eight lanes, whose rows are short, takes them from the first element on.
template <int G, class S>
struct Cut {
  static constexpr int V = VECTOR<S>;
  int head, nvec, singles;
  __device__ __forceinline__ Cut(const S *x, int n) {
    head = G < 16 ? 0 : (int)((0 - (uintptr_t)x / sizeof(S)) % V);
    head = head < n ? head : n;
    nvec = (n - head) / V;
    singles = n - nvec * V;
  }
  __device__ __forceinline__ int vector(int c) const { return head + c * V; }
  __device__ __forceinline__ int single(int i) const { return i < head ? i : nvec * V + i; }
};
// body(number of its first element, vector) over those of a row's vectors begin to end that a lane has, U of them requested before the
// first is looked at (past the last that one again: a load under a condition is waited for before the next).
template <int G, int U, class S, class B>
__device__ __forceinline__ void vectors(const Cut<G, S> &cut, const S *x, int begin, int end, int lane, B &&body) {
  const S *v = x + cut.head;
  for (int c = begin + lane; c < end; c += U * G) {
    Words raw[U];
#pragma unroll
    for (int u = 0; u < U; u++) raw[u] = load_vector(v, c + u * G < end ? c + u * G : end - 1);
#pragma unroll
    for (int u = 0; u < U; u++)
      if (c + u * G < end) body(cut.vector(c + u * G), raw[u]);
  }
}
// ... and one(number) over the single elements.
template <int G, int U, class S, class B, class E>
__device__ __forceinline__ void walk(const S *x, int n, int lane, B &&body, E &&one) {
  const Cut<G, S> cut(x, n);
  vectors<G, U>(cut, x, 0, cut.nvec, lane, body);
  for (int i = lane; i < cut.singles; i += G) one(cut.single(i));
}

template <class C>
struct Statistics {
  C peak, total, log_total, entropy;
};

// What a lane has seen of its row: the largest element, and against the reference a = reference(m) the sums
// s = sum 2^(x L - a) and t = sum 2^(x L - a) (x L - a).
template <int DT>
struct Running {
  using IO = Io<DT>;
  using C = typename IO::C;
  using S = typename IO::S;
  C m = -Bounds<C>::inf, a = Bounds<C>::low, s = 0, t = 0;
  template <int N>
  __device__ __forceinline__ void take(const C (&x)[N]) {
    C top = x[0];
#pragma unroll
    for (int j = 1; j < N; j++) top = larger(top, x[j]);
    raise(larger(m, top));
#pragma unroll
    for (int j = 0; j < N; j++) {
      const C d = fused(x[j], Bounds<C>::L, -a), p = power(d);
      s = s + p;
      t = fused(p, larger(d, Bounds<C>::none), t);  // (0 for -inf, not 0 * -inf)
    }
  }
  __device__ __forceinline__ void raise(C peak) {
    const C to = reference(peak), d = larger(a - to, Bounds<C>::none), k = power(d);
    t = fused(s, d, t) * k;
    s = s * k;
    m = peak;
    a = to;
  }
  __device__ __forceinline__ void take(Words raw) {
    C x[IO::V];
    IO::widen(raw, x);
    take(x);
  }
  __device__ __forceinline__ void take_one(S raw) {
    const C x[1] = {IO::ld(raw)};
    take(x);
  }
  // its values as the k-th of count, in shared or device memory
  __device__ __forceinline__ void store(C *at, int count) const {
    at[0] = m;
    at[count] = s;
    at[2 * count] = t;
  }
  __device__ __forceinline__ void load(const C *at, int count) {
    m = at[0];
    a = reference(m);
    s = at[count];
    t = at[2 * count];
  }
  template <int G, int U>
  __device__ __forceinline__ void take_row(const S *x, int n, int lane) {
    walk<G, U>(x, n, lane, [&](int, Words raw) { take(raw); }, [&](int i) { take_one(x[i]); });
  }
  // joined with the other lanes of a group of N
  template <int N>
  __device__ __forceinline__ void join() {
    raise(lanes_combine<N>(m, Larger<C>{}));
    s = lanes_combine<N>(s, Sum<C>{});
    t = lanes_combine<N>(t, Sum<C>{});
  }
};

// The statistics of a row by differences with its largest element, which is given: for rows that are not near.
template <int DT, int G>
__device__ __forceinline__ Statistics<typename Tr<DT>::C> far_statistics(const typename Tr<DT>::S *x, int n, int lane, typename Tr<DT>::C peak,
                                                                         typename Tr<DT>::C *lds) {
  using IO = Io<DT>;
  using C = typename IO::C;
  C sums[2] = {0, 0};
  auto take = [&](C v) {
    const C d = v - peak, p = power(d * Bounds<C>::L);
    sums[0] = sums[0] + p;
    sums[1] = fused(p, larger(d, Bounds<C>::none), sums[1]);
  };
  walk<G, 1>(x, n, lane,
             [&](int, Words raw) {
               C v[IO::V];
               IO::widen(raw, v);
#pragma unroll
               for (int j = 0; j < IO::V; j++) take(v[j]);
             },
             [&](int i) { take(IO::ld(x[i])); });
  group_combine<G>(sums, Sum<C>{}, lds);  // (NaN, from -inf - -inf, where every logit is -inf: there is no distribution)
  const C log_total = log(sums[0]);
  return {peak, sums[0], log_total, log_total - sums[1] / sums[0]};
}

// Shared memory of a group of several waves: the waves' triples, twice, so that one barrier a row will do; sums of rows that are not near.
template <class C, int G>
struct Space {
  C wave[2][G > 64 ? 3 * (G / 64) : 1], sums[G > 64 ? 2 * (G / 64) : 1];
};
// The lanes' sums joined: every lane of the group gets them. turn: 0 and 1 from one row of the block to the next.
template <int DT, int G>
__device__ __forceinline__ void join_group(Running<DT> &r, int lane, int turn, Space<typename Tr<DT>::C, G> &l) {
  r.template join<(G < 64 ? G : 64)>();
  if constexpr (G > 64) {
    constexpr int W = G / 64;
    auto *w = l.wave[turn];
    if ((lane & 63) == 0) r.store(w + (lane >> 6), W);
    __syncthreads();
    r.load(w + lane % W, W);
    r.template join<W>();
  }
}
// The statistics of row x from its sums.
template <int DT, int G>
__device__ __forceinline__ Statistics<typename Tr<DT>::C> finish(const Running<DT> &r, const typename Tr<DT>::S *x, int n, int lane,
                                                                 Space<typename Tr<DT>::C, G> &l) {
  using C = typename Tr<DT>::C;
  if (!is_near(r.m)) return far_statistics<DT, G>(x, n, lane, r.m, l.sums);
  const C lost = fused(r.m, Bounds<C>::L, -r.a);
  C total = r.s * power(-lost);
  total = total < 1 ? 1 : total;  // (the peak's own term is 1)
  const C log_total = log(total), entropy = log_total - Bounds<C>::ln2 * (r.t / r.s - lost);
  return {r.m, total, log_total, entropy < 0 ? 0 : entropy};
}

// The log probability of a row's token: one below zero is padding, one past the row names nothing.
template <int DT>
__device__ __forceinline__ typename Tr<DT>::C token_log_p(const typename Tr<DT>::S *x, int n, int token, const Statistics<typename Tr<DT>::C> &z) {
  using C = typename Tr<DT>::C;
  if (token < 0) return 0;
  if (token >= n) return (C)__builtin_nan("");
  return Io<DT>::ld(x[token]) - z.peak - z.log_total;
}
template <int DT>
__device__ __forceinline__ void give_statistics(const LogProbsArgs &a, const Places &p, const typename Tr<DT>::S *x,
                                                const Statistics<typename Tr<DT>::C> &z) {
  using C = typename Tr<DT>::C;
  if (a.o[LP_LOG_P].base) *place<C>(a, p, LP_LOG_P) = token_log_p<DT>(x, a.g.n, *place<const int32_t>(a, p, LP_TOKEN), z);
  if (a.o[LP_ENTROPY].base) *place<C>(a, p, LP_ENTROPY) = z.entropy;
  if (a.o[LP_PEAK].base) *place<C>(a, p, LP_PEAK) = z.peak;
  if (a.o[LP_TOTAL].base) *place<C>(a, p, LP_TOTAL) = z.total;
}

constexpr int group_threads(int g) { return g > 256 ? g : 256; }
constexpr int AHEAD = 4;  // vectors that a lane requests at once

template <int DT, int G>
__global__ __launch_bounds__(group_threads(G)) void log_probs_kernel(LogProbsArgs a) {
  using C = typename Tr<DT>::C;
  using S = typename Tr<DT>::S;
  constexpr int GROUPS = group_threads(G) / G;
  __shared__ Space<C, G> space;
  const int lane = threadIdx.x % G;
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * GROUPS + group_number<G, group_threads(G)>(); row < a.g.rows; row += (int64_t)gridDim.x * GROUPS, turn ^= 1) {
    Places p;
    row_starts(a.g, (uint32_t)row, a.o, p.at);
    const S *x = place<const S>(a, p, LP_X);
    Running<DT> r;
    r.template take_row<G, AHEAD>(x, a.g.n, lane);
    join_group<DT, G>(r, lane, turn, space);
    const Statistics<C> z = finish<DT, G>(r, x, a.g.n, lane, space);
    if (lane == 0) give_statistics<DT>(a, p, x, z);
  }
}

// ── the gradient ────────────────────────────────────────────────────────────
// What a row's gradient is made for.
template <class C>
struct Upstream {
  C g, g_entropy;
  int token;
};
template <class C>
__device__ __forceinline__ Upstream<C> upstream(const LogProbsArgs &a, const Places &p) {
  return {*place<const C>(a, p, LP_G), a.o[LP_G_ENTROPY].base ? *place<const C>(a, p, LP_G_ENTROPY) : 0, *place<const int32_t>(a, p, LP_TOKEN)};
}
template <int DT>
struct Gradient {
  using IO = Io<DT>;
  using C = typename IO::C;
  using S = typename IO::S;
  C peak, ref, inv_total, g, g_entropy, shift;  // inner = log p + entropy = ln2 d + shift for the exponent d
  int token;
  bool with_entropy, near;
  uint32_t there;  // all bits; none for padding without an entropy's gradient, which has zeros whatever its logits are: NaNs among them
  __device__ __forceinline__ Gradient(const LogProbsArgs &a, const Upstream<C> &up, const Statistics<C> &z) {
    peak = z.peak;
    near = is_near(peak);
    ref = reference(peak);
    const C lost = near ? fused(peak, Bounds<C>::L, -ref) : 0;
    inv_total = power(-lost) / z.total;
    token = up.token;
    g = token < 0 ? 0 : token >= a.g.n ? (C)__builtin_nan("") : up.g;
    with_entropy = a.o[LP_G_ENTROPY].base != nullptr;
    there = token < 0 && !with_entropy ? 0 : ~0u;
    g_entropy = up.g_entropy;
    shift = with_entropy ? z.entropy - z.log_total - Bounds<C>::ln2 * lost : 0;
  }
  template <bool NEAR, bool ENTROPY>
  __device__ __forceinline__ C at(C x) const {
    const C d = NEAR ? fused(x, Bounds<C>::L, -ref) : (x - peak) * Bounds<C>::L, p = power(d) * inv_total;
    return ENTROPY ? -p * fused(g_entropy, fused(larger(d, Bounds<C>::none), Bounds<C>::ln2, shift), g) : -g * p;
  }
  // Of the elements from number i of the row on.
  template <bool NEAR, bool ENTROPY>
  __device__ __forceinline__ Words vector(Words raw, int i) const {
    C v[IO::V];
    IO::widen(raw, v);
#pragma unroll
    for (int j = 0; j < IO::V; j++) v[j] = at<NEAR, ENTROPY>(v[j]);
    const unsigned j = (unsigned)(token - i);
    if (j < (unsigned)IO::V)
#pragma unroll
      for (int k = 0; k < IO::V; k++) v[k] = v[k] + ((unsigned)k == j ? g : 0);
    return IO::narrow(v) & there;
  }
  template <bool NEAR, bool ENTROPY>
  __device__ __forceinline__ S element(S x, int i) const {
    return there ? IO::st(at<NEAR, ENTROPY>(IO::ld(x)) + (i == token ? g : 0)) : S{};
  }
  // The gradient of the row's vectors begin to end, by G lanes, and of its single elements.
  template <int G, int U, bool NEAR, bool ENTROPY>
  __device__ __forceinline__ void write(const Cut<G, S> &cut, const S *x, S *out, int begin, int end, bool singles, int lane) const {
    vectors<G, U>(cut, x, begin, end, lane, [&](int i, Words raw) { store_words(element_at(out, i), vector<NEAR, ENTROPY>(raw, i)); });
    if (singles)
      for (int i = lane; i < cut.singles; i += G) out[cut.single(i)] = element<NEAR, ENTROPY>(x[cut.single(i)], cut.single(i));
  }
  template <int G, int U>
  __device__ __forceinline__ void of(const Cut<G, S> &cut, const S *x, S *out, int begin, int end, bool singles, int lane) const {
    if (near && !with_entropy) write<G, U, true, false>(cut, x, out, begin, end, singles, lane);
    else if (near) write<G, U, true, true>(cut, x, out, begin, end, singles, lane);
    else write<G, 1, false, true>(cut, x, out, begin, end, singles, lane);
  }
};

// A row's vectors are dealt out to gridDim.x groups of lanes, in equal shares.
template <int DT, int G>
__global__ __launch_bounds__(256) void log_probs_grad_kernel(LogProbsArgs a) {
  using C = typename Tr<DT>::C;
  using S = typename Tr<DT>::S;
  constexpr int GROUPS = 256 / G;
  const int lane = threadIdx.x % G;
  for (int64_t row = (int64_t)blockIdx.y * GROUPS + threadIdx.x / G; row < a.g.rows; row += (int64_t)gridDim.y * GROUPS) {
    Places p;
    row_starts(a.g, (uint32_t)row, a.o, p.at);
    Statistics<C> z{*place<const C>(a, p, LP_PEAK), *place<const C>(a, p, LP_TOTAL), 0, 0};
    if (a.o[LP_G_ENTROPY].base) {
      z.log_total = log(z.total);
      z.entropy = *place<const C>(a, p, LP_ENTROPY);
    }
    const Gradient<DT> grad(a, upstream<C>(a, p), z);
    const S *x = place<const S>(a, p, LP_X);
    const Cut<G, S> cut(x, a.g.n);
    const int share = (cut.nvec + (int)gridDim.x - 1) / (int)gridDim.x, begin = (int)blockIdx.x * share;
    grad.template of<G, AHEAD>(cut, x, place<S>(a, p, LP_D), begin, begin + share < cut.nvec ? begin + share : cut.nvec, blockIdx.x == 0, lane);
  }
}

// Statistics and gradient of a row by the same lanes, whose vectors, at most NV of a lane, stay in registers from the one to the
// other; as one has been written, the next row's is requested into its place, so that memory works while sums are taken.
template <int DT, int G, int NV>
__global__ __launch_bounds__(group_threads(G)) void log_probs_with_grad_kernel(LogProbsArgs a) {
  using IO = Io<DT>;
  using C = typename IO::C;
  using S = typename IO::S;
  constexpr int GROUPS = group_threads(G) / G;
  __shared__ Space<C, G> space;
  const int lane = threadIdx.x % G, n = a.g.n;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  int64_t row = (int64_t)blockIdx.x * GROUPS + group_number<G, group_threads(G)>();
  if (row >= a.g.rows) return;  // (whole groups; a group of several waves is the block)
  Places p;
  const S *x;
  // The gradient may go where the logits are, log_p and entropy where g and g_entropy are: the token's logit and the row's own
  // values are read here, before the lane's other logits, which the sums are made of that all lanes wait for.
  S picked, alone{};
  Upstream<C> up;
  auto begin = [&](int64_t r) {
    row_starts(a.g, (uint32_t)r, a.o, p.at);
    x = place<const S>(a, p, LP_X);
    up = upstream<C>(a, p);
    picked = x[up.token < 0 || up.token >= n ? 0 : up.token];
  };
  begin(row);
  Cut<G, S> cut(x, n);  // (at most one of its single elements is a lane's)
  auto request = [&](const Cut<G, S> &of, int v) {
    return load_vector(x + of.head, v * G + lane < of.nvec ? v * G + lane : of.nvec > 0 ? of.nvec - 1 : 0);
  };
  // (a row without a vector has fewer elements than one and is not read by vectors: then none has)
  const bool has = cut.nvec > 0;
  Words raw[NV];
  if (has)
#pragma unroll
    for (int v = 0; v < NV; v++) raw[v] = request(cut, v);
  if (lane < cut.singles) alone = x[cut.single(lane)];
  for (int turn = 0; row < a.g.rows; row += step, turn ^= 1) {
    Running<DT> r;
#pragma unroll
    for (int v = 0; v < NV; v++) {
      if (v * G + lane < cut.nvec) r.take(raw[v]);
      __builtin_amdgcn_sched_barrier(0);  // (one after the other: widened at once they need more registers)
    }
    if (lane < cut.singles) r.take_one(alone);
    join_group<DT, G>(r, lane, turn, space);
    const Statistics<C> z = finish<DT, G>(r, x, n, lane, space);
    if (lane == 0) {
      if (a.o[LP_LOG_P].base)
        *place<C>(a, p, LP_LOG_P) = up.token < 0 ? 0 : up.token >= n ? (C)__builtin_nan("") : IO::ld(picked) - z.peak - z.log_total;
      if (a.o[LP_ENTROPY].base) *place<C>(a, p, LP_ENTROPY) = z.entropy;
    }
    if constexpr (G > 64)
      if (!is_near(z.peak)) __syncthreads();  // (the walk by differences was the last to read the row)
    const Gradient<DT> grad(a, up, z);
    S *out = place<S>(a, p, LP_D);
    begin(row + step < a.g.rows ? row + step : row);  // (behind the last row its own again, for nothing)
    const Cut<G, S> next(x, n);
    auto write = [&](auto near, auto entropy) {
      constexpr bool NEAR = decltype(near)::value, ENTROPY = decltype(entropy)::value;
      if (has)
#pragma unroll
        for (int v = 0; v < NV; v++) {
          const Words d = grad.template vector<NEAR, ENTROPY>(raw[v], cut.vector(v * G + lane));
          raw[v] = request(next, v);
          if (v * G + lane < cut.nvec) store_words(element_at(out, cut.vector(v * G + lane)), d);
          __builtin_amdgcn_sched_barrier(0);
        }
      if (lane < cut.singles) {
        const S d = grad.template element<NEAR, ENTROPY>(alone, cut.single(lane));
        out[cut.single(lane)] = d;
      }
      if (lane < next.singles) alone = x[next.single(lane)];
    };
    if (grad.near && !grad.with_entropy) write(std::true_type{}, std::false_type{});
    else if (grad.near) write(std::true_type{}, std::true_type{});
    else write(std::false_type{}, std::true_type{});
    cut = next;
  }
}
// Rows longer than that are read again, out of the caches: those of float64 from 257 vectors on, which then have 1024 lanes each, many of them
// with no vector ([8192,512] float64 22 us by the kernel above, [8192,600] 156 by this one, [4096,1500] 97, [2048,4000] 70).
template <int DT, int G>
__global__ __launch_bounds__(G) void log_probs_with_grad_long_kernel(LogProbsArgs a) {
  using IO = Io<DT>;
  using C = typename IO::C;
  using S = typename IO::S;
  __shared__ Space<C, G> space;
  const int lane = threadIdx.x, n = a.g.n;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.g.rows; row += gridDim.x, turn ^= 1) {
    Places p;
    row_starts(a.g, (uint32_t)row, a.o, p.at);
    const S *x = place<const S>(a, p, LP_X);
    const Upstream<C> up = upstream<C>(a, p);
    const S picked = x[up.token < 0 || up.token >= n ? 0 : up.token];  // (first, as above)
    Running<DT> r;
    r.template take_row<G, AHEAD>(x, n, lane);
    join_group<DT, G>(r, lane, turn, space);
    const Statistics<C> z = finish<DT, G>(r, x, n, lane, space);
    if (lane == 0) {
      if (a.o[LP_LOG_P].base)
        *place<C>(a, p, LP_LOG_P) = up.token < 0 ? 0 : up.token >= n ? (C)__builtin_nan("") : IO::ld(picked) - z.peak - z.log_total;
      if (a.o[LP_ENTROPY].base) *place<C>(a, p, LP_ENTROPY) = z.entropy;
    }
    if (!is_near(z.peak)) __syncthreads();
    const Gradient<DT> grad(a, up, z);
    const Cut<G, S> cut(x, n);
    grad.template of<G, AHEAD>(cut, x, place<S>(a, p, LP_D), 0, cut.nvec, true, lane);
  }
}

// ── the most likely tokens ──────────────────────────────────────────────────
// Elements are ordered by keys: unsigned words in the order of the values, NaNs below all of them, 0 for no element; of equal keys
// the lower index comes first.
template <class C> struct KeyOf { using T = uint32_t; };
template <> struct KeyOf<double> { using T = uint64_t; };
template <class C>
__device__ __forceinline__ typename KeyOf<C>::T key_of(C x) {
  using T = typename KeyOf<C>::T;
  constexpr T sign = (T)1 << (8 * sizeof(T) - 1);
  const T u = __builtin_bit_cast(T, x + 0);  // (-0 equals 0)
  return x != x ? 1 : (u & sign) ? ~u : u | sign;
}
template <class C>
__device__ __forceinline__ C value_of(typename KeyOf<C>::T k) {
  using T = typename KeyOf<C>::T;
  constexpr T sign = (T)1 << (8 * sizeof(T) - 1);
  return k == 1 ? (C)__builtin_nan("") : __builtin_bit_cast(C, (k & sign) ? k & ~sign : ~k);
}
template <class T>
struct Highest {
  __device__ __forceinline__ T operator()(T a, T b) const { return a > b ? a : b; }
};

constexpr int TOP_MAX = 64;  // alternatives

template <int DT, int G>
struct TopSpace {
  using T = typename KeyOf<typename Tr<DT>::C>::T;
  static constexpr int PLACES = G > 64 ? 1024 : 512, LANES = G > 64 ? 5 * TOP_MAX : 64;  // of candidates; of lanes that may hold them
  T key[PLACES];
  uint32_t index[PLACES], lane[LANES], few[64];
  T lane_key[LANES], few_key[64], low[G / 64];
  int part[G / 64], lanes, found;
};

// Of each of W waves' lanes the k / W, rounded up, with the largest elements: the least of those k bounds the k-th largest element
// of the row from below, and only lanes whose largest reaches it hold candidates: one or two times k in a row without
// order, of which, where they are few, the k largest are found. All lanes together look through those lanes' elements. Ties (a row of equal logits, a vocabulary that is banned but for a few tokens) can make candidates of the
// whole row: then what lies above the bound is taken, and of what equals it the first in the row. A row whose large elements
// gather in a few lanes, and one with a NaN, has its k-th largest found bit by bit, a walk for each.
template <int DT, int G>
struct Top {
  using IO = Io<DT>;
  using C = typename IO::C;
  using S = typename IO::S;
  using T = typename KeyOf<C>::T;
  static constexpr int V = IO::V, W = G / 64, PLACES = TopSpace<DT, G>::PLACES, LANES = TopSpace<DT, G>::LANES;
  // A key has so many bits that tell elements apart, above some that do not (float16 has 19, bfloat16 16).
  static constexpr int BITS = sizeof(S) == 2 ? 20 : 8 * (int)sizeof(T), SPARE = 8 * (int)sizeof(T) - BITS;
  const S *x;
  int n, k;
  const Cut<G, S> cut;
  TopSpace<DT, G> &l;
  const int lane = threadIdx.x, wave = threadIdx.x >> 6;
  T mine = 0;

  __device__ __forceinline__ Top(const S *row, int length, int top, TopSpace<DT, G> &space) : x(row), n(length), k(top), cut(row, length), l(space) {}

  // give(place, key, index) for the k largest of the first m entries of the list. A wave's lanes hold an entry each and count the
  // larger ones. Of 65 to 256 entries each of several waves takes its share, an entry at a time, against four that each lane holds (one
  // wave by itself: 59 us for 64 of [20,260] float32, 20 as follows). Of more, the k-th is found first, bit by bit of the key, and
  // of the index where entries tie there.
  template <class F>
  __device__ __forceinline__ void rank(int m, F &&give) const {
    if (W > 1 && m > 64 && m <= 256) {
      constexpr int Q = 4;
      T key[Q];
      uint32_t index[Q];
#pragma unroll
      for (int q = 0; q < Q; q++) {
        const int j = q * 64 + (lane & 63);
        key[q] = j < m ? l.key[j] : 0;
        index[q] = j < m ? l.index[j] : ~0u;  // (before nothing)
      }
      for (int i = wave; i < m; i += W) {
        const T mine = l.key[i];
        const uint32_t at = l.index[i];
        int place = 0;
#pragma unroll
        for (int q = 0; q < Q; q++)
          if (q * 64 < m) place += __popcll(__ballot(key[q] > mine || (key[q] == mine && index[q] < at)));
        if ((lane & 63) == 0 && place < k) give(place, mine, at);
      }
      return;
    }
    if (wave != 0) return;
    T key = 0;
    uint32_t index = 0;
    int count = m;
    if (m <= 64) {
      if (lane < m) {
        key = l.key[lane];
        index = l.index[lane];
      }
    } else {
      auto number = [&](auto &&is) {
        int c = 0;
        for (int j = lane; j - lane < m; j += 256) {
          T e[4];
#pragma unroll
          for (int q = 0; q < 4; q++) e[q] = l.key[j + q * 64 < m ? j + q * 64 : m - 1] >> SPARE;
#pragma unroll
          for (int q = 0; q < 4; q++) c += __popcll(__ballot(j + q * 64 < m && is(e[q], j + q * 64)));
        }
        return c;
      };
      T bound = 0;
      for (int bit = BITS - 1; bit >= 0; bit--) {
        const T next = bound | (T)1 << bit;
        if (number([&](T e, int) { return e >= next; }) >= k) bound = next;
      }
      const int above = number([&](T e, int) { return e > bound; }), least = number([&](T e, int) { return e >= bound; });
      uint32_t last = ~0u;  // of those at the bound the first ones, up to this index
      if (least > k) {
        last = 0;
        for (int bit = 31 - __builtin_clz(n); bit >= 0; bit--) {
          const uint32_t next = last | 1u << bit;
          if (above + number([&](T e, int j) { return e == bound && l.index[j] < next; }) < k) last = next;
        }
      }
      count = 0;
      for (int j = lane; j - lane < m; j += 64) {
        const T e = j < m ? l.key[j] : 0;
        const uint32_t i = j < m ? l.index[j] : ~0u;
        const bool is = j < m && (e >> SPARE > bound || (e >> SPARE == bound && i <= last));
        const uint64_t all = __ballot(is);
        if (is) {
          const int place = count + __popcll(all & (((uint64_t)1 << lane) - 1));
          l.few_key[place] = e;
          l.few[place] = i;
        }
        count += __popcll(all);
      }
      __builtin_amdgcn_wave_barrier();
      if (lane < count) {
        key = l.few_key[lane];
        index = l.few[lane];
      }
    }
    int place = 0;
    for (int j = 0; j < count; j++) {
      const T other = lane_value(key, j);
      place += other > key || (other == key && (uint32_t)__builtin_amdgcn_readlane((int)index, j) < index);
    }
    if (lane < count && place < k) give(place, key, index);
  }
  __device__ __forceinline__ static uint32_t lane_value(uint32_t v, int j) { return (uint32_t)__builtin_amdgcn_readlane((int)v, j); }
  __device__ __forceinline__ static uint64_t lane_value(uint64_t v, int j) {
    return (uint64_t)lane_value((uint32_t)(v >> 32), j) << 32 | lane_value((uint32_t)v, j);
  }
  __device__ __forceinline__ void offer(S raw, int i, T least) {
    const T key = key_of(IO::ld(raw));
    if (key >= least) {
      const int at = atomicAdd(&l.found, 1);
      if (at < PLACES) {
        l.key[at] = key;
        l.index[at] = (uint32_t)i;
      }
    }
  }
  __device__ __forceinline__ void offer(Words raw, int i, T least) {
    struct Elements { S x[V]; } e = __builtin_bit_cast(Elements, raw);
#pragma unroll
    for (int j = 0; j < V; j++) offer(e.x[j], i + j, least);
  }
  // The k-th largest of the keys of a wave's lanes, down to the bits that tell them apart.
  __device__ __forceinline__ static T wave_kth(T key, int k) {
    T kth = 0;
#pragma unroll
    for (int bit = BITS + SPARE - 1; bit >= SPARE; bit--) {
      const T next = kth | (T)1 << bit;
      if (__popcll(__ballot(key >= next)) >= k) kth = next;
    }
    return kth;
  }
  // Before the barrier of the statistics: the wave's part in the bound. Waves that are not full of vectors take no part in it; of a
  // row that one wave holds every lane with an element is looked at.
  __device__ __forceinline__ void begin(C seen) {
    const int nvec = cut.nvec, full = nvec <= 64 ? 0 : nvec / 64 < W ? nvec / 64 : W;
    mine = lane < nvec || lane < cut.singles ? key_of(seen) : 0;
    T most = full ? ~(T)0 : 1;
    if (wave < full) {
      const int share = (k + full - 1) / full;
      if (share > 8) {
        most = wave_kth(mine, share);
      } else {
        T left = mine;
        for (int r = 0; r < share; r++) {
          most = lanes_combine<64>(left, Highest<T>{});
          const uint64_t have = __ballot(left == most);
          if ((lane & 63) == __builtin_ctzll(have)) left = 0;
        }
      }
    }
    if ((lane & 63) == 0) l.low[wave] = most;
    if (lane == 0) l.lanes = l.found = 0;
  }
  // Every element of key `least` or more of the row onto the list, which may want more places than it has.
  __device__ __forceinline__ int collect(T least) {
    __syncthreads();
    if (lane == 0) l.found = 0;
    __syncthreads();
    walk<G, 1>(x, n, lane, [&](int i, Words raw) { offer(raw, i, least); }, [&](int i) { offer(x[i], i, least); });
    __syncthreads();
    return l.found;
  }
  // The k-th largest key of the row.
  __device__ __forceinline__ T by_bits() {
    T bound = 0;
    for (int bit = 8 * (int)sizeof(T) - 1; bit >= 0; bit--) {
      const T next = bound | (T)1 << bit;
      int count[1] = {0};
      walk<G, 1>(x, n, lane,
                 [&](int, Words raw) {
                   struct Elements { S x[V]; } e = __builtin_bit_cast(Elements, raw);
#pragma unroll
                   for (int j = 0; j < V; j++) count[0] += key_of(IO::ld(e.x[j])) >= next;
                 },
                 [&](int i) { count[0] += key_of(IO::ld(x[i])) >= next; });
      group_combine<G>(count, Sum<int>{}, l.part);
      if (count[0] >= k) bound = next;
    }
    return bound;
  }
  // The first elements of the row that equal the bound, from place `at` of the list on, up to k.
  __device__ __forceinline__ void first_equal(T bound, int at) {
    for (int base = 0; at < k && base < n; base += G) {
      const bool hit = base + lane < n && key_of(IO::ld(x[base + lane])) == bound;
      const uint64_t hits = __ballot(hit);
      __syncthreads();
      if ((lane & 63) == 0) l.part[wave] = __popcll(hits);
      __syncthreads();
      int place = at + __popcll(hits & (((uint64_t)1 << (lane & 63)) - 1));
#pragma unroll
      for (int w = 0; w < W; w++) {
        if (w < wave) place += l.part[w];
        at += l.part[w];
      }
      if (hit && place < k) {
        l.key[place] = bound;
        l.index[place] = (uint32_t)(base + lane);
      }
    }
    __syncthreads();
  }
  // After the barrier of the statistics: the list holds the k largest elements, and others; how many.
  __device__ __forceinline__ int candidates(bool ordered) {
    T bound = 0;
    int found = PLACES + 1;
    if (ordered) {
      bound = l.low[0];
#pragma unroll
      for (int w = 1; w < W; w++) bound = l.low[w] < bound ? l.low[w] : bound;
      if (mine >= bound) {
        const int at = atomicAdd(&l.lanes, 1);
        if (at < LANES) {
          l.lane[at] = (uint32_t)lane;
          l.lane_key[at] = mine;
        }
      }
      __syncthreads();
      int lanes = l.lanes;
      const uint32_t *which = l.lane;
      if (lanes <= 64) {  // each wave by itself finds the k-th largest of them, down to the bits that a 16-bit dtype has
        const int i = lane & 63;
        const T key = i < lanes ? l.lane_key[i] : 0;
        const T kth = wave_kth(key, k);
        if (kth > bound) bound = kth;
        const uint64_t reach = __ballot(i < lanes && key >= bound);
        if (reach >> i & 1) l.few[__popcll(reach & (((uint64_t)1 << i) - 1))] = l.lane[i];  // (the same of every wave)
        lanes = __popcll(reach);
        which = l.few;
      }
      if (lanes <= LANES) {
        const int each = (cut.nvec + G - 1) / G;
        for (int w = lane; w < lanes * each; w += G) {
          const int c = (w / lanes) * G + (int)which[w % lanes];
          if (c < cut.nvec) offer(load_vector(x + cut.head, c), cut.vector(c), bound);
        }
        if (lane < cut.singles) offer(x[cut.single(lane)], cut.single(lane), bound);
        __syncthreads();
        found = l.found;
        if (found <= PLACES) return found;
      }
      found = collect(bound + 1);
    }
    if (found > PLACES) {
      bound = by_bits();
      found = collect(bound + 1);  // fewer than k
    }
    if (found >= k) return found;
    first_equal(bound, found);
    return k;
  }
  __device__ __forceinline__ void write(int found, const Statistics<C> &z, C *log_p, int32_t *tokens) const {
    rank(found, [&](int place, T key, uint32_t index) {
      log_p[place] = value_of<C>(key) - z.peak - z.log_total;
      tokens[place] = (int32_t)index;
    });
  }
};

template <int DT, int G>
__global__ __launch_bounds__(G) void log_probs_top_kernel(LogProbsArgs a) {
  using C = typename Tr<DT>::C;
  using S = typename Tr<DT>::S;
  __shared__ Space<C, G> space;
  __shared__ TopSpace<DT, G> list;
  const int lane = threadIdx.x, n = a.g.n;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.g.rows; row += gridDim.x, turn ^= 1) {
    Places p;
    row_starts(a.g, (uint32_t)row, a.o, p.at);
    const S *x = place<const S>(a, p, LP_X);
    Top<DT, G> top(x, n, a.top, list);
    Running<DT> r;
    r.template take_row<G, AHEAD>(x, n, lane);
    top.begin(r.m);
    join_group<DT, G>(r, lane, turn, space);
    if constexpr (G == 64) __syncthreads();  // (what begin wrote is there)
    const Statistics<C> z = finish<DT, G>(r, x, n, lane, space);
    if (lane == 0) give_statistics<DT>(a, p, x, z);
    top.write(top.candidates(z.total == z.total), z, place<C>(a, p, LP_TOP_LOG_P), place<int32_t>(a, p, LP_TOP_TOKEN));
    __syncthreads();  // the list is free for the next row
  }
}

// ── few long rows ───────────────────────────────────────────────────────────
// Rows that would leave most of the chip idle are cut into parts, a block to each: a part's sums and its own most likely tokens, in their
// order, go to memory, and a block for each row joins them. (A row of 200000 float32 logits 17.1 us whole, 7.1 in parts; statistics and
// gradient of [20,150000] 26 and 15 us.)
constexpr int PART_LANES = 256, JOIN_LANES = 1024, PARTS_MAX = 16;
struct Parts {
  void *sums;       // [rows][3][parts]
  void *keys;       // [rows][parts][top]
  uint32_t *index;  // [rows][parts][top]
  void *values;     // [5][rows]: peak, total, entropy, g and g_entropy for the gradient; null: not wanted
  int parts, share;  // vectors of a part; the last has the elements behind the last vector too
};
template <int DT>
__global__ __launch_bounds__(PART_LANES) void log_probs_parts_kernel(LogProbsArgs a, Parts q) {
  using C = typename Tr<DT>::C;
  using S = typename Tr<DT>::S;
  using T = typename KeyOf<C>::T;
  constexpr int G = PART_LANES, V = VECTOR<S>;
  __shared__ Space<C, G> space;
  __shared__ TopSpace<DT, G> list;
  const int lane = threadIdx.x, part = blockIdx.x;
  const int64_t row = blockIdx.y;
  Places p;
  row_starts(a.g, (uint32_t)row, a.o, p.at);
  const int first = part * q.share * V, n = part + 1 == q.parts ? a.g.n - first : q.share * V;
  const S *x = place<const S>(a, p, LP_X) + first;
  Top<DT, G> top(x, n, a.top, list);
  Running<DT> r;
  r.template take_row<G, AHEAD>(x, n, lane);
  if (a.top) top.begin(r.m);
  join_group<DT, G>(r, lane, 0, space);
  if (lane == 0) r.store(reinterpret_cast<C *>(q.sums) + row * 3 * q.parts + part, q.parts);
  if (!a.top) return;
  const int64_t at = (row * q.parts + part) * a.top;
  top.rank(top.candidates(r.s == r.s), [&](int place, T key, uint32_t index) {
    reinterpret_cast<T *>(q.keys)[at + place] = key;
    q.index[at + place] = index + (uint32_t)first;
  });
}
template <int DT>
__global__ __launch_bounds__(JOIN_LANES) void log_probs_join_kernel(LogProbsArgs a, Parts q) {
  using C = typename Tr<DT>::C;
  using S = typename Tr<DT>::S;
  using T = typename KeyOf<C>::T;
  constexpr int G = JOIN_LANES;
  __shared__ Space<C, G> space;
  __shared__ TopSpace<DT, G> list;
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  Places p;
  row_starts(a.g, (uint32_t)row, a.o, p.at);
  const S *x = place<const S>(a, p, LP_X);
  // The row's k-th is bounded from below by any part's k-th, and by the least of the parts' k / parts-th, rounded up.
  const T *keys = reinterpret_cast<const T *>(q.keys) + row * q.parts * a.top;
  const int offered = q.parts * a.top, part = lane % PARTS_MAX;
  T bound = 0;
  if (a.top) {
    const bool has = part < q.parts;
    const T kth = lanes_combine<PARTS_MAX>(has ? keys[(part + 1) * a.top - 1] : 0, Highest<T>{});
    const T share = ~lanes_combine<PARTS_MAX>(has ? ~keys[part * a.top + (a.top - 1) / q.parts] : 0, Highest<T>{});
    bound = kth > share ? kth : share;
  }
  if (lane == 0) list.found = 0;
  __syncthreads();
  if (lane < offered && keys[lane] >= bound) {  // (at most 16 * 64 = JOIN_LANES, and as many places)
    const int at = atomicAdd(&list.found, 1);
    list.key[at] = keys[lane];
    list.index[at] = q.index[row * offered + lane];
  }
  Running<DT> r;
  if (part < q.parts) r.load(reinterpret_cast<const C *>(q.sums) + row * 3 * q.parts + part, q.parts);
  r.template join<PARTS_MAX>();
  const Statistics<C> z = finish<DT, G>(r, x, a.g.n, lane, space);
  if (lane == 0) {
    if (C *v = reinterpret_cast<C *>(q.values)) {
      const Upstream<C> up = upstream<C>(a, p);  // (log_p and entropy may go where they are)
      v[row] = z.peak;
      v[a.g.rows + row] = z.total;
      v[2 * a.g.rows + row] = z.entropy;
      v[3 * a.g.rows + row] = up.g;
      v[4 * a.g.rows + row] = up.g_entropy;
    }
    give_statistics<DT>(a, p, x, z);
  }
  __syncthreads();
  Top<DT, G>(x, a.g.n, a.top, list).write(list.found, z, place<C>(a, p, LP_TOP_LOG_P), place<int32_t>(a, p, LP_TOP_TOKEN));
}

// ── host side ───────────────────────────────────────────────────────────────
// Of rows that are not cut: vectors, and, with alternatives, whose search goes by the element, elements.
constexpr int WHOLE_VECTORS = 8192, WHOLE_TOP = 72 << 10;
constexpr int64_t MOST_LANES = (int64_t)1 << 31;  // of a launch, which numbers them in 32 bits; groups go on to further rows

// A row's lanes: eight where its vectors are no more, a wave up to four vectors a lane, a block of four waves up to eight, then one
// of eight waves ([8192,50257] bfloat16: 141 us, 145 with four waves, 211 with sixteen, of which only two blocks are on a unit and
// wait for each other's phases; five alternatives of [2048,50257] float32: 75, 81 and 97 us).
template <int DT, class F>
void by_length(int n, F &&f) {
  constexpr int V = VECTOR<typename Tr<DT>::S>;
  if (n <= 8 * V) f(std::integral_constant<int, 8>{});
  else if (n <= 4 * 64 * V) f(std::integral_constant<int, 64>{});
  else if (n <= 8 * 256 * V) f(std::integral_constant<int, 256>{});
  else f(std::integral_constant<int, 512>{});
}
dim3 row_blocks(const LogProbsArgs &a, int threads, int group) {
  const int64_t groups = threads / group;
  return dim3((unsigned)std::min((a.g.rows + groups - 1) / groups, MOST_LANES / threads));
}
// How many parts a row is cut into; 1: not at all. Two launches more and what the parts pass on have to pay (eight rows of bfloat16, whole
// and in parts: statistics of 50257 elements 6.5 and 7.0 us, of 80000 8.6 and 6.8; with their gradient 11.7 and 10.7, 14.5 and 10.6;
// with 20 alternatives 11.3 and 15.6, 14.0 and 13.3, of 131000 17.7 and 14.9; of 50257 float32 12.2 and 14.2, of a row of 200000 22.9
// and 14.4), and a block for every row has to leave three quarters of the units idle. At that border of 64 and 65 rows the two are even at
// 80000 float32 (statistics 10.1 in parts, 10.3 whole; with their gradient 18.0, 17.3; with 20 alternatives 19.1, 17.2); longer rows would gain
// from parts beyond it (150000: 11.7 and 16.9; 24.7 and 30.4; 22.0 and 28.1).
template <int DT>
int parts_of(nxh_context *ctx, const LogProbsArgs &a) {
  const int64_t units = ctx->compute_units > 0 ? ctx->compute_units : 256, nvec = a.g.n / VECTOR<typename Tr<DT>::S>;
  if (nvec <= WHOLE_VECTORS || (a.top && a.g.n <= WHOLE_TOP) || a.g.rows * 4 > units) return 1;
  return (int)std::min<int64_t>(std::min<int64_t>(PARTS_MAX, 2 * units / a.g.rows), nvec / (2 * PART_LANES));
}
// The statistics and most likely tokens of rows in parts. values: room for [5][rows], or null.
template <int DT>
int launch_parts(nxh_context *ctx, const LogProbsArgs &a, int parts, void *values) {
  using C = typename Tr<DT>::C;
  const int nvec = a.g.n / VECTOR<typename Tr<DT>::S>;
  Parts q;
  q.share = (nvec + parts - 1) / parts;
  q.parts = (nvec + q.share - 1) / q.share;
  q.values = values;
  const size_t sums = (size_t)a.g.rows * 3 * q.parts * sizeof(C), list = (size_t)a.g.rows * q.parts * a.top;
  void *space = nullptr;
  if (int rc = nxh_alloc_locked(ctx, sums + list * (sizeof(typename KeyOf<C>::T) + 4), &space)) return rc;
  q.sums = space;
  q.keys = (char *)space + sums;
  q.index = (uint32_t *)((char *)q.keys + list * sizeof(typename KeyOf<C>::T));
  hipLaunchKernelGGL((log_probs_parts_kernel<DT>), dim3((unsigned)q.parts, (unsigned)a.g.rows), dim3(PART_LANES), 0, ctx->stream, a, q);
  hipLaunchKernelGGL((log_probs_join_kernel<DT>), dim3((unsigned)a.g.rows), dim3(JOIN_LANES), 0, ctx->stream, a, q);
  nxh_free_locked(ctx, space);  // (the stream orders its next use behind these launches)
  return NXH_OK;
}
template <int DT>
int launch_score(nxh_context *ctx, const LogProbsArgs &a) {
  if (const int parts = parts_of<DT>(ctx, a); parts > 1) return launch_parts<DT>(ctx, a, parts, nullptr);
  by_length<DT>(a.g.n, [&](auto group) {
    constexpr int G = decltype(group)::value;
    if (!a.top) {
      hipLaunchKernelGGL((log_probs_kernel<DT, G>), row_blocks(a, group_threads(G), G), dim3(group_threads(G)), 0, ctx->stream, a);
    } else {
      constexpr int B = G > 64 ? G : 64;
      hipLaunchKernelGGL((log_probs_top_kernel<DT, B>), row_blocks(a, B, B), dim3(B), 0, ctx->stream, a);
    }
  });
  return NXH_OK;
}
template <int DT>
int launch_grad(nxh_context *ctx, const LogProbsArgs &a) {
  constexpr int V = VECTOR<typename Tr<DT>::S>;
  auto go = [&](auto group) {
    constexpr int G = decltype(group)::value;
    const int parts = std::max(1, (a.g.n / V + G * AHEAD - 1) / (G * AHEAD));  // (at most 2^14)
    const int64_t rows = (a.g.rows + 256 / G - 1) / (256 / G);
    const dim3 grid((unsigned)parts, (unsigned)std::min(rows, std::min<int64_t>(65535, MOST_LANES / 256 / parts)));
    hipLaunchKernelGGL((log_probs_grad_kernel<DT, G>), grid, dim3(256), 0, ctx->stream, a);
  };
  if (a.g.n <= 8 * V) go(std::integral_constant<int, 8>{});
  else if (a.g.n <= 4 * 64 * V) go(std::integral_constant<int, 64>{});
  else go(std::integral_constant<int, 256>{});
  return NXH_OK;
}

template <int DT>
int launch_with_grad(nxh_context *ctx, const LogProbsArgs &a) {
  using C = typename Tr<DT>::C;
  constexpr int V = VECTOR<typename Tr<DT>::S>;
  if (const int parts = parts_of<DT>(ctx, a); parts > 1) {
    void *values = nullptr;
    if (int rc = nxh_alloc_locked(ctx, (size_t)a.g.rows * 5 * sizeof(C), &values)) return rc;
    int rc = launch_parts<DT>(ctx, a, parts, values);
    if (!rc) {
      LogProbsArgs b = a;
      constexpr int which[] = {LP_PEAK, LP_TOTAL, LP_ENTROPY, LP_G, LP_G_ENTROPY};
      for (int k = 0; k < (a.o[LP_G_ENTROPY].base ? 5 : 4); k++) {
        RowOperand &o = b.o[which[k]];
        o.base = (const char *)values + (size_t)k * a.g.rows * sizeof(C);
        int64_t stride = 1;
        for (int d = a.g.nouter - 1; d >= 0; d--) {
          o.stride[d] = stride;
          stride *= a.g.oshape[d];
        }
      }
      rc = launch_grad<DT>(ctx, b);
    }
    nxh_free_locked(ctx, values);
    return rc;
  }
  const int64_t units = ctx->compute_units > 0 ? ctx->compute_units : 256;
  auto go = [&](auto group, auto vectors) {
    constexpr int G = decltype(group)::value, T = group_threads(G), NV = decltype(vectors)::value;
    // As many blocks as the chip has room for, but for 256 lanes with eight vectors: their 84 registers (float32; 16-bit dtypes 94) leave
    // a unit room for five blocks, of which it gets four. (512 lanes: two; 1024: one.)
    const int64_t blocks = std::min((a.g.rows + T / G - 1) / (T / G), units * ((NV == 8 ? 1024 : 2048) / T));
    hipLaunchKernelGGL((log_probs_with_grad_kernel<DT, G, NV>), dim3((unsigned)blocks), dim3(T), 0, ctx->stream, a);
  };
  const int nvec = a.g.n / V;
  if (nvec <= 8) {
    go(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
    return NXH_OK;
  }
  if (nvec <= 4 * 64) {
    go(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
    return NXH_OK;
  }
  if constexpr (DT != NXH_F64) {  // (float64 has no registers for more)
    std::integral_constant<int, 8> eight;
    if (nvec <= 8 * 256) go(std::integral_constant<int, 256>{}, eight);
    else if (nvec <= 8 * 512) go(std::integral_constant<int, 512>{}, eight);
    else if (nvec <= 8 * 1024) go(std::integral_constant<int, 1024>{}, eight);
    if (nvec <= 8 * 1024) return NXH_OK;
  }
  hipLaunchKernelGGL((log_probs_with_grad_long_kernel<DT, 1024>), row_blocks(a, 1024, 1024), dim3(1024), 0, ctx->stream, a);
  return NXH_OK;
}
// What the three calls check alike; false in *go where there is nothing to launch.
int prepare(const char *op, LogProbsArgs &a, const nxh_tensor *logits, const nxh_tensor *tokens, bool *go) {
  int rc = NXH_OK;
  *go = false;
  if ((rc = rows_geometry(op, logits, a.g))) return rc;
  if (!float_dtype_ok(logits->dtype)) return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
  if ((rc = row_values_ok(op, tokens, logits, NXH_I32))) return rc;
  for (auto &o : a.o) row_operand(nullptr, o);
  a.top = 0;
  if (a.g.rows == 0) return NXH_OK;
  if (a.g.n == 0) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_EMPTY_REDUCE);
  if (!unit_stride(logits)) return nxh_fail(NXH_FAILURE, op, "rows must be contiguous");
  row_operand(logits, a.o[LP_X]);
  row_value_operand(tokens, a.o[LP_TOKEN]);
  *go = true;
  return NXH_OK;
}
// A value for each row, that is read or written.
int value_operand(const char *op, LogProbsArgs &a, int k, const nxh_tensor *t, const nxh_tensor *logits, bool written) {
  if (!t) return NXH_OK;
  if (int rc = row_values_ok(op, t, logits, statistics_dtype(logits->dtype))) return rc;
  if (written)
    if (int rc = out_rows_ok(op, t)) return rc;
  row_value_operand(t, a.o[k]);
  return NXH_OK;
}
int gradient_operand(const char *op, LogProbsArgs &a, const nxh_tensor *out, const nxh_tensor *logits) {
  if (int rc = same_shape(op, out, logits)) return rc;
  if (int rc = out_rows_ok(op, out)) return rc;
  if (out->dtype != logits->dtype) return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
  if (a.g.rows > 0 && a.g.n > 0 && !unit_stride(out)) return nxh_fail(NXH_FAILURE, op, "rows must be contiguous");
  row_operand(out, a.o[LP_D]);
  return NXH_OK;
}
int start(nxh_context *ctx, const char *op, const char *path, LogProbsArgs &a) {
  merge_outer_dims(a.g, {&a.o[0], &a.o[1], &a.o[2], &a.o[3], &a.o[4], &a.o[5], &a.o[6], &a.o[7], &a.o[8], &a.o[9], &a.o[10]});
  NXH_HIP(op, hipSetDevice(ctx->device));
  nxh_set_path(path);
  return NXH_OK;
}
#define LP_BY_DTYPE(dt, f)                                                \
  ((dt) == NXH_F32 ? f<NXH_F32>(ctx, a) : (dt) == NXH_BF16 ? f<NXH_BF16>(ctx, a) : (dt) == NXH_F16 ? f<NXH_F16>(ctx, a) : f<NXH_F64>(ctx, a))

}  // namespace

NXH_EXPORT int nxh_log_probs(nxh_context *ctx, const nxh_tensor *log_p, const nxh_tensor *entropy, const nxh_tensor *peak,
                             const nxh_tensor *total, const nxh_tensor *top_log_p, const nxh_tensor *top_tokens,
                             const nxh_tensor *logits, const nxh_tensor *tokens) {
  NXH_DEFER_TOUCH(ctx, 6, log_p, entropy, peak, total, top_log_p, top_tokens, logits, tokens);
  const char *op = "log_probs";
  if (!ctx || !logits || !tokens || (!top_log_p) != (!top_tokens)) return nxh_fail(NXH_INVALID_ARGUMENT, op, "null argument");
  int rc = NXH_OK;
  for (const nxh_tensor *t : {log_p, entropy, peak, total, top_log_p, top_tokens, logits, tokens})
    if (t && (rc = nxh_check_tensor(op, t))) return rc;
  LogProbsArgs a;
  bool go;
  if ((rc = prepare(op, a, logits, tokens, &go))) return rc;
  const nxh_tensor *values[] = {log_p, entropy, peak, total};
  for (int k = 0; k < 4; k++)
    if ((rc = value_operand(op, a, LP_LOG_P + k, values[k], logits, true))) return rc;
  if (top_log_p) {
    const int last = logits->ndim - 1;
    if (top_log_p->dtype != statistics_dtype(logits->dtype) || top_tokens->dtype != NXH_I32)
      return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
    if ((rc = same_shape(op, top_log_p, top_tokens)) || (rc = out_rows_ok(op, top_log_p)) || (rc = out_rows_ok(op, top_tokens))) return rc;
    if (top_log_p->ndim != logits->ndim) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
    for (int d = 0; d < last; d++)
      if (top_log_p->shape[d] != logits->shape[d]) return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
    const int64_t top = top_log_p->shape[last];
    if (top > TOP_MAX) return nxh_fail(NXH_FAILURE, op, "more than 64 alternatives");
    if (top > logits->shape[last]) return nxh_fail(NXH_INVALID_ARGUMENT, op, "more alternatives than a row has elements");
    if (top > 0 && (!unit_stride(top_log_p) || !unit_stride(top_tokens))) return nxh_fail(NXH_FAILURE, op, "rows must be contiguous");
    row_operand(top_log_p, a.o[LP_TOP_LOG_P]);
    row_operand(top_tokens, a.o[LP_TOP_TOKEN]);
    a.top = (int)top;
  }
  if (!go) return NXH_OK;
  std::lock_guard<std::mutex> guard(ctx->mu);
  if ((rc = start(ctx, op, a.top ? "log_probs_top" : "log_probs", a))) return rc;
  if ((rc = LP_BY_DTYPE(logits->dtype, launch_score))) return rc;
  NXH_HIP(op, hipGetLastError());
  return NXH_OK;
}

NXH_EXPORT int nxh_log_probs_grad(nxh_context *ctx, const nxh_tensor *out, const nxh_tensor *g, const nxh_tensor *logits,
                                  const nxh_tensor *tokens, const nxh_tensor *peak, const nxh_tensor *total,
                                  const nxh_tensor *g_entropy, const nxh_tensor *entropy) {
  NXH_DEFER_TOUCH(ctx, 1, out, g, logits, tokens, peak, total, g_entropy, entropy);
  const char *op = "log_probs_grad";
  if (!ctx || !out || !g || !logits || !tokens || !peak || !total || (!g_entropy) != (!entropy))
    return nxh_fail(NXH_INVALID_ARGUMENT, op, "null argument");
  int rc = NXH_OK;
  for (const nxh_tensor *t : {out, g, logits, tokens, peak, total, g_entropy, entropy})
    if (t && (rc = nxh_check_tensor(op, t))) return rc;
  LogProbsArgs a;
  bool go;
  if ((rc = prepare(op, a, logits, tokens, &go)) || (rc = gradient_operand(op, a, out, logits))) return rc;
  const std::pair<int, const nxh_tensor *> values[] = {{LP_G, g}, {LP_PEAK, peak}, {LP_TOTAL, total}, {LP_G_ENTROPY, g_entropy}, {LP_ENTROPY, entropy}};
  for (auto &v : values)
    if ((rc = value_operand(op, a, v.first, v.second, logits, false))) return rc;
  if (!go) return NXH_OK;
  std::lock_guard<std::mutex> guard(ctx->mu);
  if ((rc = start(ctx, op, "log_probs_grad", a))) return rc;
  if ((rc = LP_BY_DTYPE(logits->dtype, launch_grad))) return rc;
  NXH_HIP(op, hipGetLastError());
  return NXH_OK;
}

NXH_EXPORT int nxh_log_probs_with_grad(nxh_context *ctx, const nxh_tensor *log_p, const nxh_tensor *entropy, const nxh_tensor *out,
                                       const nxh_tensor *g, const nxh_tensor *logits, const nxh_tensor *tokens,
                                       const nxh_tensor *g_entropy) {
  NXH_DEFER_TOUCH(ctx, 3, log_p, entropy, out, g, logits, tokens, g_entropy);
  const char *op = "log_probs_with_grad";
  if (!ctx || !out || !g || !logits || !tokens) return nxh_fail(NXH_INVALID_ARGUMENT, op, "null argument");
  int rc = NXH_OK;
  for (const nxh_tensor *t : {log_p, entropy, out, g, logits, tokens, g_entropy})
    if (t && (rc = nxh_check_tensor(op, t))) return rc;
  LogProbsArgs a;
  bool go;
  if ((rc = prepare(op, a, logits, tokens, &go)) || (rc = gradient_operand(op, a, out, logits))) return rc;
  if ((rc = value_operand(op, a, LP_LOG_P, log_p, logits, true)) || (rc = value_operand(op, a, LP_ENTROPY, entropy, logits, true)) ||
      (rc = value_operand(op, a, LP_G, g, logits, false)) || (rc = value_operand(op, a, LP_G_ENTROPY, g_entropy, logits, false)))
    return rc;
  if (!go) return NXH_OK;
  std::lock_guard<std::mutex> guard(ctx->mu);
  if ((rc = start(ctx, op, "log_probs_with_grad", a))) return rc;
  if ((rc = LP_BY_DTYPE(logits->dtype, launch_with_grad))) return rc;
  NXH_HIP(op, hipGetLastError());
  return NXH_OK;
}
