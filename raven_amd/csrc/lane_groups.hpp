// lane_groups.hpp — what the training kernels over rows share (layer_norm.hip,
// layer_norm_grad.hip, log_probs.hip): a row belongs to a group of G lanes, several groups to a
// wave (G < 64), one wave, or a whole block of G / 64 waves; its elements come in vectors of 16
// bytes at whatever alignment the row has.
#pragma once

#include <type_traits>

#include "nxh_common.hpp"

namespace {

template <class S>
constexpr int VECTOR = 16 / (int)sizeof(S);

// Sixteen bytes of a row, as words: elements are taken out where they are used (kept as an array of 16-bit elements between a load
// and its use, the compiler takes them apart at the load, which waits for it).
typedef uint32_t Words __attribute__((ext_vector_type(4)));
// A 16-byte access needs no more than an element's alignment, so rows of odd lengths and views that
// start anywhere are read and written as wide as aligned ones.
template <class S>
__device__ __forceinline__ Words load_words(const S *p) {
  Words w;
  __builtin_memcpy(&w, p, sizeof w);
  return w;
}
template <class S>
__device__ __forceinline__ void store_words(S *p, Words w) {
  __builtin_memcpy(p, &w, sizeof w);
}

// Element i of a row, by an offset of 32 bits (a row has at most 2^27 bytes): beside a row that all lanes share it is one register, for
// every operand the same.
template <class S>
__device__ __forceinline__ S *element_at(S *row, int i) {
  using Byte = std::conditional_t<std::is_const<S>::value, const char, char>;
  return reinterpret_cast<S *>(reinterpret_cast<Byte *>(row) + (uint32_t)i * (uint32_t)sizeof(S));
}

// Vector c of a row.
template <class S>
__device__ __forceinline__ Words load_vector(const S *row, int c) {
  return load_words(element_at(row, c * VECTOR<S>));
}

// What elements are computed as, and back, one or a vector at a time. float16 and bfloat16 take the hardware's conversions, which
// round to nearest, ties to even, and keep a NaN a NaN; the primitives' keep its payload too, at some ten instructions an
// element of float16.
template <int DT>
struct Io {
  using S = typename Tr<DT>::S;
  using C = typename Tr<DT>::C;
  static constexpr int V = VECTOR<S>;
  __device__ __forceinline__ static C ld(S s) {
    if constexpr (DT == NXH_F16) return (float)__builtin_bit_cast(_Float16, s);
    else return Tr<DT>::ld(s);
  }
  __device__ __forceinline__ static S st(C c) {
    if constexpr (DT == NXH_F16) {
      asm("" : "+v"(c));  // (a product folded into the conversion would lose the sign of zero)
      return __builtin_bit_cast(uint16_t, (_Float16)c);
    } else {
      return Tr<DT>::st(c);
    }
  }
  __device__ __forceinline__ static void widen(Words w, C (&x)[V]) {
    if constexpr (sizeof(S) == 2) {
#pragma unroll
      for (int k = 0; k < 4; k++) {
        if constexpr (DT == NXH_BF16) {
          x[2 * k] = u2f(w[k] << 16);
          x[2 * k + 1] = u2f(w[k] & 0xffff0000u);
        } else {
          x[2 * k] = ld((S)(w[k] & 0xffffu));
          x[2 * k + 1] = ld((S)(w[k] >> 16));
        }
      }
    } else {
      struct Elements { C x[V]; } e = __builtin_bit_cast(Elements, w);
#pragma unroll
      for (int j = 0; j < V; j++) x[j] = e.x[j];
    }
  }
  __device__ __forceinline__ static Words narrow(const C (&x)[V]) {
    Words w;
    if constexpr (sizeof(S) == 2) {
#pragma unroll
      for (int k = 0; k < 4; k++) {
        if constexpr (DT == NXH_BF16) w[k] = f32x2_to_bf16x2(x[2 * k], x[2 * k + 1]);
        else w[k] = (uint32_t)st(x[2 * k]) | (uint32_t)st(x[2 * k + 1]) << 16;
      }
    } else {
      struct Elements { C x[V]; } e;
#pragma unroll
      for (int j = 0; j < V; j++) e.x[j] = x[j];
      w = __builtin_bit_cast(Words, e);
    }
    return w;
  }
  __device__ __forceinline__ static Words all(C c) {
    C x[V];
#pragma unroll
    for (int j = 0; j < V; j++) x[j] = c;
    return narrow(x);
  }
};

// Vector c of a row of n elements. WHOLE: n is a number of vectors. RAGGED: it is none and more than one; the last vector is the
// row's last V elements, of which it has the first in common with the one before it: they are loaded, computed and stored
// twice, with equal results, and belong to sums once. SHORT: less than a vector, which is taken element by element.
enum Rows { WHOLE, RAGGED, SHORT };
template <int V, Rows R>
__device__ __forceinline__ int vec_start(int c, int n) {
  return R != RAGGED || (c + 1) * V <= n ? c * V : n - V;
}
// Whether element j of vector c belongs to it.
template <int V, Rows R>
__device__ __forceinline__ bool vec_owns(int c, int j, int n) {
  return R == WHOLE ? true : R == SHORT ? j < n : j >= c * V - vec_start<V, R>(c, n);
}
template <Rows R, class S>
__device__ __forceinline__ Words load_part(const S *row, int c, int n) {
  constexpr int V = VECTOR<S>;
  if constexpr (R != SHORT) return load_words(element_at(row, vec_start<V, R>(c, n)));
  struct Elements { S x[V]; } e;
#pragma unroll
  for (int j = 0; j < V; j++) e.x[j] = row[j < n ? j : 0];
  return __builtin_bit_cast(Words, e);
}
template <Rows R, class S>
__device__ __forceinline__ void store_part(S *row, int c, int n, Words w) {
  constexpr int V = VECTOR<S>;
  if constexpr (R != SHORT) {
    store_words(element_at(row, vec_start<V, R>(c, n)), w);
  } else {
    struct Elements { S x[V]; } e = __builtin_bit_cast(Elements, w);
#pragma unroll
    for (int j = 0; j < V; j++)
      if (j < n) row[j] = e.x[j];
  }
}
// Only what the vector owns: for results that replace what other lanes may not have read yet.
template <class S>
__device__ __forceinline__ void store_own(S *row, int c, int n, Words w) {
  constexpr int V = VECTOR<S>;
  if ((c + 1) * V <= n) {
    store_words(element_at(row, c * V), w);
    return;
  }
  struct Elements { S x[V]; } e = __builtin_bit_cast(Elements, w);
#pragma unroll
  for (int j = 0; j < V; j++)
    if (vec_owns<V, RAGGED>(c, j, n)) row[vec_start<V, RAGGED>(c, n) + j] = e.x[j];
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
// f over K values of each of a group's lanes at once; every lane gets the same bits. A group of several waves is the whole block and
// meets in `lds` (K * G / 64 values), of which each lane reads one wave's: all of sixteen waves' would be as many registers.
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
    for (int k = 0; k < K; k++) v[k] = lanes_combine<W>(lds[(threadIdx.x % W) * K + k], f);
  }
}

// Which of a block's T / G groups a lane belongs to. Groups of whole waves have it, and the addresses that follow from it, in
// scalar registers.
template <int G, int T>
__device__ __forceinline__ int group_number() {
  if constexpr (G == T) return 0;
  else if constexpr (G >= 64) return __builtin_amdgcn_readfirstlane((int)threadIdx.x / G);
  else return (int)threadIdx.x / G;
}

template <class C>
struct Sum {
  __device__ __forceinline__ C operator()(C a, C b) const { return a + b; }
};

__device__ __forceinline__ float fused(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fused(double a, double b, double c) { return __builtin_fma(a, b, c); }

}  // namespace
