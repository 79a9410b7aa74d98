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
// logits once; the gradient once more in and out.

#include <type_traits>
#include <utility>

#include "lane_groups.hpp"
#include "rows.hpp"
#include "softmax_math.hpp"

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

// e^x for x <= 0. The statistics of 16-bit logits take the hardware's exponential alone: its error, and that of the product
// in front of it, are some 2^-22 of a term, and no term of the gradient keeps more than 11 bits. float32 logits have both corrected.
template <int DT>
struct Exp {
  __device__ __forceinline__ static float of(float x) { return __builtin_amdgcn_exp2f(x * 0x1.715476p+0f); }
};
template <>
struct Exp<NXH_F32> {
  __device__ __forceinline__ static float of(float x) { return exp_nonpositive(x); }
};
template <>
struct Exp<NXH_F64> {
  __device__ __forceinline__ static double of(double x) { return exp(x); }
};
__device__ __forceinline__ float larger(float a, float b) { return __builtin_fmaxf(a, b); }  // (a NaN is passed over: the sums have it)
__device__ __forceinline__ double larger(double a, double b) { return __builtin_fmax(a, b); }
template <class C>
struct Larger {
  __device__ __forceinline__ C operator()(C a, C b) const { return larger(a, b); }
};
// The lowest finite value, which a lane starts from (differences with it are no NaN), and a difference whose exponential is 0.
template <class C> struct Bounds;
template <> struct Bounds<float> { static constexpr float lowest = -0x1.fffffep+127f, far = -200.0f, inf = __builtin_inff(); };
template <> struct Bounds<double> { static constexpr double lowest = -0x1.fffffffffffffp+1023, far = -2000.0, inf = __builtin_inf(); };

template <class C>
struct Statistics {
  C peak, total, log_total, entropy;
};

// What a lane has seen of its row.
template <int DT>
struct Running {
  using TX = Tr<DT>;
  using C = typename TX::C;
  using S = typename TX::S;
  C m = Bounds<C>::lowest, s = 0, t = 0;
  C seen = -Bounds<C>::inf;  // the largest element, which m is not where all are -inf
  template <int W>
  __device__ __forceinline__ void take(const Vec<S, W> &raw) {
    C x[W], top = TX::ld(raw.v[0]);
    x[0] = top;
#pragma unroll
    for (int j = 1; j < W; j++) {
      x[j] = TX::ld(raw.v[j]);
      top = larger(top, x[j]);
    }
    seen = larger(seen, top);
    raise(larger(m, top));
#pragma unroll
    for (int j = 0; j < W; j++) {
      const C d = x[j] - m, p = Exp<DT>::of(d);
      s = s + p;
      t = fused(p, larger(d, Bounds<C>::far), t);  // (0 for -inf, not 0 * -inf)
    }
  }
  // the sums against another peak, no lower than m
  __device__ __forceinline__ void raise(C peak) {
    const C d = larger(m - peak, Bounds<C>::far), k = Exp<DT>::of(d);
    t = fused(s, d, t) * k;
    s = s * k;
    m = peak;
  }
};

// body(vector number) over the vectors of a row that a lane has: numbers lane, lane + G, ... four requested before the first is
// looked at; then tail(index) for the single elements behind the last whole vector, one to a lane.
template <int V, int G, class S, class B, class E>
__device__ __forceinline__ void walk(const S *x, int n, int lane, B &&body, E &&tail) {
  constexpr int U = 4;
  const int nvec = n / V;
  int c = lane;
  for (; c + (U - 1) * G < nvec; c += U * G) {
    Vec<S, V> raw[U];
#pragma unroll
    for (int u = 0; u < U; u++) raw[u] = load_vec<V>(x + (int64_t)(c + u * G) * V);
#pragma unroll
    for (int u = 0; u < U; u++) body(c + u * G, raw[u]);
  }
  for (; c < nvec; c += G) body(c, load_vec<V>(x + (int64_t)c * V));
  if (nvec * V + lane < n) tail(nvec * V + lane);
}

template <int DT, int G>
__device__ __forceinline__ Statistics<typename Tr<DT>::C> statistics(const typename Tr<DT>::S *x, int n, int lane, typename Tr<DT>::C *lds,
                                                                     typename Tr<DT>::C &seen) {
  using C = typename Tr<DT>::C;
  using S = typename Tr<DT>::S;
  Running<DT> r;
  walk<VECTOR<S>, G>(x, n, lane, [&](int, const Vec<S, VECTOR<S>> &raw) { r.take(raw); }, [&](int i) { r.take(load_vec<1>(x + i)); });
  seen = r.seen;
  C m[1] = {r.m};
  group_combine<G>(m, Larger<C>{}, lds);
  r.raise(m[0]);
  C sums[2] = {r.s, r.t};
  group_combine<G>(sums, Sum<C>{}, lds);
  Statistics<C> z{m[0], sums[0], 0, 0};
  if (z.total == 0) {  // every logit is -inf: there is no distribution
    z.peak = -Bounds<C>::inf;
    z.total = __builtin_nan("");
  }
  z.log_total = log(z.total);
  z.entropy = z.log_total - sums[1] / z.total;
  return z;
}

// The log probability of a row's token: one below zero is padding, one past the row names nothing.
template <int DT>
__device__ __forceinline__ typename Tr<DT>::C token_log_p(const typename Tr<DT>::S *x, int n, int token, const Statistics<typename Tr<DT>::C> &z) {
  using C = typename Tr<DT>::C;
  if (token < 0) return 0;
  if (token >= n) return (C)__builtin_nan("");
  return Tr<DT>::ld(x[token]) - z.peak - z.log_total;
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

template <int DT, int G>
__global__ __launch_bounds__(group_threads(G)) void log_probs_kernel(LogProbsArgs a) {
  using C = typename Tr<DT>::C;
  using S = typename Tr<DT>::S;
  constexpr int GROUPS = group_threads(G) / G;
  __shared__ C lds[G > 64 ? 2 * (G / 64) : 1];
  const int lane = threadIdx.x % G;
  for (int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / G; row < a.g.rows; row += (int64_t)gridDim.x * GROUPS) {
    Places p;
    row_starts(a.g, (uint32_t)row, a.o, p.at);
    const S *x = place<const S>(a, p, LP_X);
    C seen;
    const Statistics<C> z = statistics<DT, G>(x, a.g.n, lane, lds, seen);
    if (lane == 0) give_statistics<DT>(a, p, x, z);
  }
}

// ── the gradient ────────────────────────────────────────────────────────────
template <int DT>
struct Gradient {
  using TX = Tr<DT>;
  using C = typename TX::C;
  using S = typename TX::S;
  Statistics<C> z;
  C inv_total, g, g_entropy;
  int token;
  bool with_entropy;
  __device__ __forceinline__ Gradient(const LogProbsArgs &a, const Places &p, const Statistics<C> &s) : z(s) {
    inv_total = 1 / z.total;
    token = *place<const int32_t>(a, p, LP_TOKEN);
    g = token < 0 ? 0 : token >= a.g.n ? (C)__builtin_nan("") : *place<const C>(a, p, LP_G);
    with_entropy = a.o[LP_G_ENTROPY].base != nullptr;
    g_entropy = with_entropy ? *place<const C>(a, p, LP_G_ENTROPY) : 0;
  }
  __device__ __forceinline__ C at(C x) const {
    const C d = x - z.peak, p = Exp<DT>::of(d) * inv_total;
    if (!with_entropy) return -g * p;
    return -p * fused(g_entropy, larger(d, Bounds<C>::far) - z.log_total + z.entropy, g);
  }
  template <int W>
  __device__ __forceinline__ Vec<S, W> of(const Vec<S, W> &raw, int first) const {
    C d[W];
#pragma unroll
    for (int j = 0; j < W; j++) d[j] = at(TX::ld(raw.v[j]));
    if ((unsigned)(token - first) < (unsigned)W)
#pragma unroll
      for (int j = 0; j < W; j++)
        if (first + j == token) d[j] = d[j] + g;
    Vec<S, W> o;
#pragma unroll
    for (int j = 0; j < W; j++) o.v[j] = TX::st(d[j]);
    return o;
  }
};

// A row's vectors are dealt out to gridDim.x groups of lanes.
constexpr int GRAD_VECTORS = 4;  // of a lane
template <int DT, int G>
__global__ __launch_bounds__(256) void log_probs_grad_kernel(LogProbsArgs a) {
  using C = typename Tr<DT>::C;
  using S = typename Tr<DT>::S;
  constexpr int V = VECTOR<S>, GROUPS = 256 / G;
  const int lane = threadIdx.x % G, n = a.g.n;
  const int first = blockIdx.x * G * GRAD_VECTORS;
  const int part = n - first * V < G * GRAD_VECTORS * V ? n - first * V : G * GRAD_VECTORS * V;
  for (int64_t row = (int64_t)blockIdx.y * GROUPS + threadIdx.x / G; row < a.g.rows; row += (int64_t)gridDim.y * GROUPS) {
    Places p;
    row_starts(a.g, (uint32_t)row, a.o, p.at);
    const S *x = place<const S>(a, p, LP_X) + (int64_t)first * V;
    S *out = place<S>(a, p, LP_D) + (int64_t)first * V;
    Statistics<C> z{*place<const C>(a, p, LP_PEAK), *place<const C>(a, p, LP_TOTAL), 0, 0};
    if (a.o[LP_G_ENTROPY].base) {
      z.log_total = log(z.total);
      z.entropy = *place<const C>(a, p, LP_ENTROPY);
    }
    Gradient<DT> grad(a, p, z);
    walk<V, G>(x, part, lane, [&](int c, const Vec<S, V> &raw) { store_vec<V>(out + (int64_t)c * V, grad.of(raw, (first + c) * V)); },
               [&](int i) { store_vec<1>(out + i, grad.of(load_vec<1>(x + i), first * V + i)); });
  }
}

// Statistics and gradient of a row by the same lanes: the second walk finds the row in the caches.
template <int DT, int G>
__global__ __launch_bounds__(group_threads(G)) void log_probs_with_grad_kernel(LogProbsArgs a) {
  using C = typename Tr<DT>::C;
  using S = typename Tr<DT>::S;
  constexpr int V = VECTOR<S>, GROUPS = group_threads(G) / G;
  __shared__ C lds[G > 64 ? 2 * (G / 64) : 1];
  const int lane = threadIdx.x % G, n = a.g.n;
  for (int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / G; row < a.g.rows; row += (int64_t)gridDim.x * GROUPS) {
    Places p;
    row_starts(a.g, (uint32_t)row, a.o, p.at);
    const S *x = place<const S>(a, p, LP_X);
    S *out = place<S>(a, p, LP_D);
    C seen;
    const Statistics<C> z = statistics<DT, G>(x, n, lane, lds, seen);
    if (lane == 0) give_statistics<DT>(a, p, x, z);
    // (the gradient may go where the logits are: the token's logit has been read by then)
    if constexpr (G > 64) __syncthreads();
    else __builtin_amdgcn_wave_barrier();
    Gradient<DT> grad(a, p, z);
    walk<V, G>(x, n, lane, [&](int c, const Vec<S, V> &raw) { store_vec<V>(out + (int64_t)c * V, grad.of(raw, c * V)); },
               [&](int i) { store_vec<1>(out + i, grad.of(load_vec<1>(x + i), i)); });
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

constexpr int TOP_MAX = 64, TOP_CANDIDATES = 1024;

template <int DT, int G>
struct TopSpace {
  using T = typename KeyOf<typename Tr<DT>::C>::T;
  T key[TOP_CANDIDATES];
  uint32_t index[TOP_CANDIDATES];
  T low[G / 64], cut;
  int part[G / 64], count;
};

// The k-th largest of the lanes' largest elements bounds the k-th largest of the row from below, and only lanes
// whose largest reaches it hold candidates: some k of them in a row without order, which walk their elements once more. Ties
// (a row of equal logits, a vocabulary that is banned but for a few tokens) can make candidates of the whole row: then what lies
// above the bound is taken, and of what equals it the first in the row. A row whose large elements gather in a few lanes, and one with a
// NaN, has its k-th largest found bit by bit, a walk for each.
template <int DT, int G>
__device__ __forceinline__ void top_tokens(const typename Tr<DT>::S *x, int n, int k, typename Tr<DT>::C seen, const Statistics<typename Tr<DT>::C> &z,
                                           TopSpace<DT, G> &l, typename Tr<DT>::C *log_p, int32_t *tokens) {
  using TX = Tr<DT>;
  using C = typename TX::C;
  using S = typename TX::S;
  using T = typename KeyOf<C>::T;
  constexpr int V = VECTOR<S>, W = G / 64;
  const int lane = threadIdx.x, wave = lane >> 6;
  const int nvec = n / V;
  const T mine = lane < nvec || nvec * V + lane < n ? key_of(seen) : 0;
  // puts what `wanted` says of this lane's elements on the list, which may want more places than it has
  auto collect = [&](bool look, auto &&wanted) {
    __syncthreads();
    if (lane == 0) l.count = 0;
    __syncthreads();
    auto offer = [&](S raw, int i) {
      const T key = key_of(TX::ld(raw));
      if (wanted(key)) {
        const int at = atomicAdd(&l.count, 1);
        if (at < TOP_CANDIDATES) {
          l.key[at] = key;
          l.index[at] = (uint32_t)i;
        }
      }
    };
    if (look)
      walk<V, G>(x, n, lane,
                 [&](int c, const Vec<S, V> &raw) {
#pragma unroll
                   for (int j = 0; j < V; j++) offer(raw.v[j], c * V + j);
                 },
                 [&](int i) { offer(x[i], i); });
    __syncthreads();
    return l.count;
  };
  T bound = 0;
  int found = TOP_CANDIDATES + 1;
  bool by_bits = !(z.total == z.total), ties = by_bits;
  if (!by_bits) {
    // Lanes that can be among the k largest: each wave's first k / W, rounded up, already are k.
    const int rounds = (k + W - 1) / W;
    __syncthreads();
    if (rounds <= 4) {
      T left = mine, most = 0;
      for (int r = 0; r < rounds; r++) {
        most = lanes_combine<64>(left, Highest<T>{});
        const uint64_t have = __ballot(left == most);
        if ((lane & 63) == __builtin_ctzll(have)) left = 0;
      }
      if ((lane & 63) == 0) l.low[wave] = most;
    } else if ((lane & 63) == 0) {
      l.low[wave] = 0;
    }
    if (lane == 0) l.count = 0;
    __syncthreads();
    T low = l.low[0];
#pragma unroll
    for (int w = 1; w < W; w++) low = l.low[w] < low ? l.low[w] : low;
    if (mine >= low) l.key[atomicAdd(&l.count, 1)] = mine;
    __syncthreads();
    const int m = l.count;
    if (lane < m) {
      int before = 0;
      for (int j = 0; j < m; j++) before += l.key[j] > l.key[lane] || (l.key[j] == l.key[lane] && j < lane);
      if (before == k - 1) l.cut = l.key[lane];
    }
    __syncthreads();
    bound = l.cut;
    if (__syncthreads_count(mine >= bound) <= 4 * k + 64) found = collect(mine >= bound, [&](T key) { return key >= bound; });
    if (found > TOP_CANDIDATES) {
      ties = true;
      found = collect(mine > bound, [&](T key) { return key > bound; });
      by_bits = found > TOP_CANDIDATES;
    }
  }
  if (by_bits) {
    bound = 0;
    for (int bit = 8 * (int)sizeof(T) - 1; bit >= 0; bit--) {
      const T next = bound | (T)1 << bit;
      int count[1] = {0};
      walk<V, G>(x, n, lane,
                 [&](int, const Vec<S, V> &raw) {
#pragma unroll
                   for (int j = 0; j < V; j++) count[0] += key_of(TX::ld(raw.v[j])) >= next;
                 },
                 [&](int i) { count[0] += key_of(TX::ld(x[i])) >= next; });
      group_combine<G>(count, Sum<int>{}, l.part);
      if (count[0] >= k) bound = next;
    }
    found = collect(true, [&](T key) { return key > bound; });  // fewer than k
  }
  if (ties && found < k) {  // the first of the row's elements that equal the bound
    int at = found;
    for (int base = 0; at < k && base < n; base += G) {
      const bool hit = base + lane < n && key_of(TX::ld(x[base + lane])) == bound;
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
    found = k;
    __syncthreads();
  }
  for (int i = lane; i < found; i += G) {
    const T key = l.key[i];
    const uint32_t index = l.index[i];
    int before = 0;
    for (int j = 0; j < found; j++) before += l.key[j] > key || (l.key[j] == key && l.index[j] < index);
    if (before < k) {
      log_p[before] = value_of<C>(key) - z.peak - z.log_total;
      tokens[before] = (int32_t)index;
    }
  }
  __syncthreads();  // the list is free for the next row
}

template <int DT, int G>
__global__ __launch_bounds__(G) void log_probs_top_kernel(LogProbsArgs a) {
  using C = typename Tr<DT>::C;
  using S = typename Tr<DT>::S;
  __shared__ C lds[2 * (G / 64)];
  __shared__ TopSpace<DT, G> space;
  for (int64_t row = blockIdx.x; row < a.g.rows; row += gridDim.x) {
    Places p;
    row_starts(a.g, (uint32_t)row, a.o, p.at);
    const S *x = place<const S>(a, p, LP_X);
    C seen;
    const Statistics<C> z = statistics<DT, G>(x, a.g.n, threadIdx.x, lds, seen);
    if (threadIdx.x == 0) give_statistics<DT>(a, p, x, z);
    top_tokens<DT, G>(x, a.g.n, a.top, seen, z, space, place<C>(a, p, LP_TOP_LOG_P), place<int32_t>(a, p, LP_TOP_TOKEN));
  }
}

// ── host side ───────────────────────────────────────────────────────────────
constexpr int64_t MOST_LANES = (int64_t)1 << 31;  // of a launch, which numbers them in 32 bits; groups go on to further rows

// A row's lanes: eight where its vectors are no more, a wave up to four vectors a lane, then a block of four or of sixteen waves.
template <int DT, class F>
void by_length(int n, F &&f) {
  constexpr int V = VECTOR<typename Tr<DT>::S>;
  if (n <= 8 * V) f(std::integral_constant<int, 8>{});
  else if (n <= 4 * 64 * V) f(std::integral_constant<int, 64>{});
  else if (n <= 4 * 256 * V) f(std::integral_constant<int, 256>{});
  else f(std::integral_constant<int, 1024>{});
}
dim3 row_blocks(const LogProbsArgs &a, int threads, int group) {
  const int64_t groups = threads / group;
  return dim3((unsigned)std::min((a.g.rows + groups - 1) / groups, MOST_LANES / threads));
}
template <int DT>
void launch_score(nxh_context *ctx, const LogProbsArgs &a) {
  by_length<DT>(a.g.n, [&](auto group) {
    constexpr int G = decltype(group)::value;
    if (!a.top) {
      hipLaunchKernelGGL((log_probs_kernel<DT, G>), row_blocks(a, group_threads(G), G), dim3(group_threads(G)), 0, ctx->stream, a);
    } else {
      constexpr int B = group_threads(G);
      hipLaunchKernelGGL((log_probs_top_kernel<DT, B>), row_blocks(a, B, B), dim3(B), 0, ctx->stream, a);
    }
  });
}
template <int DT>
void launch_with_grad(nxh_context *ctx, const LogProbsArgs &a) {
  by_length<DT>(a.g.n, [&](auto group) {
    constexpr int G = decltype(group)::value;
    hipLaunchKernelGGL((log_probs_with_grad_kernel<DT, G>), row_blocks(a, group_threads(G), G), dim3(group_threads(G)), 0, ctx->stream, a);
  });
}
template <int DT>
void launch_grad(nxh_context *ctx, const LogProbsArgs &a) {
  constexpr int V = VECTOR<typename Tr<DT>::S>;
  auto go = [&](auto group) {
    constexpr int G = decltype(group)::value;
    const int share = G * GRAD_VECTORS * V, parts = (a.g.n + share - 1) / share;  // (at most 2^14 parts)
    const int64_t rows = (a.g.rows + 256 / G - 1) / (256 / G);
    const dim3 grid((unsigned)parts, (unsigned)std::min(rows, std::min<int64_t>(65535, MOST_LANES / 256 / parts)));
    hipLaunchKernelGGL((log_probs_grad_kernel<DT, G>), grid, dim3(256), 0, ctx->stream, a);
  };
  if (a.g.n <= 8 * V) go(std::integral_constant<int, 8>{});
  else if (a.g.n <= 4 * 64 * V) go(std::integral_constant<int, 64>{});
  else go(std::integral_constant<int, 256>{});
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
#define LP_BY_DTYPE(dt, f)                       \
  do {                                           \
    if ((dt) == NXH_F32) f<NXH_F32>(ctx, a);     \
    else if ((dt) == NXH_BF16) f<NXH_BF16>(ctx, a); \
    else if ((dt) == NXH_F16) f<NXH_F16>(ctx, a);   \
    else f<NXH_F64>(ctx, a);                     \
  } while (0)

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
  LP_BY_DTYPE(logits->dtype, launch_score);
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
  LP_BY_DTYPE(logits->dtype, launch_grad);
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
  LP_BY_DTYPE(logits->dtype, launch_with_grad);
  NXH_HIP(op, hipGetLastError());
  return NXH_OK;
}
