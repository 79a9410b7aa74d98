// lane_groups.hpp — what the training kernels over rows share (layer_norm.hip,
// layer_norm_grad.hip, log_probs.hip): a row belongs to a group of G lanes, several groups to a
// wave (G < 64), one wave, or a whole block of G / 64 waves; its elements come in vectors of 16
// bytes at whatever alignment the row has.
#pragma once

#include "nxh_common.hpp"

namespace {

template <class S>
constexpr int VECTOR = 16 / (int)sizeof(S);

template <class S, int V>
struct Vec {
  S v[V];
};
// A 16-byte access needs no more than an element's alignment, so rows of odd lengths and views that
// start anywhere are read and written as wide as aligned ones.
template <int V, class S>
__device__ __forceinline__ Vec<S, V> load_vec(const S *p) {
  Vec<S, V> x;
  __builtin_memcpy(&x, p, sizeof(S) * V);
  return x;
}
template <int V, class S>
__device__ __forceinline__ void store_vec(S *p, const Vec<S, V> &x) {
  __builtin_memcpy(p, &x, sizeof(S) * V);
}
// Vector c of a row of n elements. RAGGED: the last one may reach past the row; what is not there reads as `fill`.
template <int V, bool RAGGED, class S>
__device__ __forceinline__ Vec<S, V> load_part(const S *row, int c, int n, S fill) {
  if (!RAGGED || (c + 1) * V <= n) return load_vec<V>(row + (int64_t)c * V);
  Vec<S, V> x;
#pragma unroll
  for (int j = 0; j < V; j++) {
    x.v[j] = fill;
    if (c * V + j < n) x.v[j] = row[(int64_t)c * V + j];
  }
  return x;
}
template <int V, bool RAGGED, class S>
__device__ __forceinline__ void store_part(S *row, int c, int n, const Vec<S, V> &x) {
  if (!RAGGED || (c + 1) * V <= n) {
    store_vec<V>(row + (int64_t)c * V, x);
    return;
  }
#pragma unroll
  for (int j = 0; j < V; j++)
    if (c * V + j < n) row[(int64_t)c * V + j] = x.v[j];
}

// ── exchanges between lanes ─────────────────────────────────────────────────
// The word of lane ^ D for D = 1, 2, 8; for D = 4 the word of a lane of the other half of eight.
// Register moves of the vector unit: no trip through LDS.
template <int D>
__device__ __forceinline__ uint32_t dpp_word(uint32_t v) {
  static_assert(D == 1 || D == 2 || D == 4 || D == 8, "within a row of sixteen lanes");
  constexpr int ctrl = D == 1 ? 0xB1 : D == 2 ? 0x4E : D == 4 ? 0x141 : 0x128;
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xF, 0xF, false);
}
// f(value of the lower half of each 2 D lanes, value of the upper half)
template <int D, class C, class F>
__device__ __forceinline__ C combine_step(C v, F f) {
  constexpr int W = (int)sizeof(C) / 4;
  struct Words { uint32_t w[W]; };
  const Words a = __builtin_bit_cast(Words, v);
  Words x = a, y = a;
#pragma unroll
  for (int i = 0; i < W; i++) {
    if constexpr (D == 32) {
      const auto p = __builtin_amdgcn_permlane32_swap(a.w[i], a.w[i], false, false);
      x.w[i] = p[0];
      y.w[i] = p[1];
    } else if constexpr (D == 16) {
      const auto p = __builtin_amdgcn_permlane16_swap(a.w[i], a.w[i], false, false);
      x.w[i] = p[0];
      y.w[i] = p[1];
    } else {
      y.w[i] = dpp_word<D>(a.w[i]);
    }
  }
  return f(__builtin_bit_cast(C, x), __builtin_bit_cast(C, y));
}
// f over the G <= 64 lanes of a group, f commutative; every lane gets the result.
template <int G, class C, class F>
__device__ __forceinline__ C lanes_combine(C v, F f) {
  if constexpr (G >= 2) v = combine_step<1>(v, f);
  if constexpr (G >= 4) v = combine_step<2>(v, f);
  if constexpr (G >= 8) v = combine_step<4>(v, f);  // (lanes of one half of eight hold the same by now)
  if constexpr (G >= 16) v = combine_step<8>(v, f);
  if constexpr (G >= 32) v = combine_step<16>(v, f);
  if constexpr (G >= 64) v = combine_step<32>(v, f);
  return v;
}
// f over K values of each of a group's lanes at once. A group of several waves is the whole block and meets in
// `lds` (K * G / 64 values); the waves' results are taken in order, so every lane has the same bits.
template <int G, int K, class C, class F>
__device__ __forceinline__ void group_combine(C (&v)[K], F f, C *lds) {
#pragma unroll
  for (int k = 0; k < K; k++) v[k] = lanes_combine<(G < 64 ? G : 64)>(v[k], f);
  if constexpr (G > 64) {
    constexpr int W = G / 64;
    __syncthreads();  // what lds held before has been read
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; k++) lds[(threadIdx.x >> 6) * K + k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; k++) {
      C s = lds[k];
#pragma unroll
      for (int w = 1; w < W; w++) s = f(s, lds[w * K + k]);
      v[k] = s;
    }
  }
}

template <class C>
struct Sum {
  __device__ __forceinline__ C operator()(C a, C b) const { return a + b; }
};

__device__ __forceinline__ float fused(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fused(double a, double b, double c) { return __builtin_fma(a, b, c); }

}  // namespace
