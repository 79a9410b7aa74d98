// attention_grad.hip — nxh_attention_grad: the gradients of nxh_attention_train, whose probabilities are made again
// from the scores and each row's lse. With g what flows back into out, over the pairs that the mask leaves
//   p_ij = e^(scale q_i . k_j - lse_i),  delta_i = g_i . out_i,  ds_ij = p_ij (g_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij g_i
// the last two over all query heads that share a head of keys and values. Two launches: the first has a query a
// lane (delta, which it leaves for the second, and dq), the second a key a lane (dk, dv). Both make p and ds, seven
// products in place of five: what a single walk would have to add up between blocks needs atomics, whose order
// changes results, or S x S values in memory, which cost more than two products. Equal calls give equal bits.
//
// delta starts the accumulators of the products g . v (negated), so ds is one multiplication. p and ds are rounded
// to 16 bits for the products that take them (float32: as they are); all sums are float32. In float16 p is 32 times
// as large, where 2^-14 is the smallest number with all its bits: probabilities of long rows and their differences
// lie below; a result is scaled back in its last multiplication.
//
// What bounds it: the matrix instructions of heads of 128, of which seven products take 7/5 of what the formulas have ([1,16,8192,128]
// bfloat16 causal 1049 to 1075 us, 640 to 655 TFLOP/s of five products, 895 to 917 of seven); of heads of 64 the vector unit beside them ([8,12,1024,64] 34 us
// dq and 47 dk, dv: matrix instructions are 40 % of the second's cycles); in float32 the matrix instructions ([3,6,777,80] with a mask
// 165 to 174 us).

#include "attention_tiles.hpp"

namespace {

// log2 of what p is multiplied by.
template <class EL>
constexpr float LIFT = EL::F32 || EL::BF16 ? 0.0f : 5.0f;
template <class EL>
constexpr float UNLIFT = EL::F32 || EL::BF16 ? 1.0f : 0.03125f;

// A row's lse as the exponent takes it: -inf, a probability of 0, for rows without keys and those past the end.
template <class EL>
__device__ __forceinline__ float exponent_of(float lse) {
  return lse == -INF ? -INF : __builtin_fmaf(-lse, LOG2E, LIFT<EL>);
}

// Blocks of four waves. KW = 1: each has 32 queries of 128. KW = 2: two share 32 queries, each takes every other 32 keys of a
// tile, and their sums are added at the end: twice the blocks, where there are few.
template <class EL, int DP, int KW, bool MASK>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu((EL::F32 || KW == 2 || MASK) && DP > (EL::F32 && (KW == 2 || MASK) ? 64 : 96) ? 1 : 2))) void attention_grad_queries_kernel(AttentionArgs a) {
  using S = typename EL::S;
  constexpr int KEYS = EL::F32 || DP > 64 ? 32 * KW : 64, SUBS = KEYS / 32 / KW, QUERIES = 128 / KW, OT = DP / 32;
  using T = Tile<EL, DP, KEYS, 4>;
  constexpr int STAGE = 2 * T::SIZE, RING = 3 * STAGE <= 80 * 1024 ? 3 : 2, AHEAD = RING - 1;  // tiles on their way
  __shared__ __attribute__((aligned(1024))) unsigned char stages[RING * STAGE];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c32 = lane & 31;
  const int pair = wave / KW, part = wave % KW;
  const uint32_t heads = (uint32_t)a.batch * (uint32_t)a.heads;
  const int tile = a.tiles - 1 - (int)(blockIdx.x / heads);
  const int bh = (int)(blockIdx.x % heads), b = bh / a.heads, h = bh % a.heads, hk = h / (a.heads / a.kv_heads);
  const int keys = keys_of(a, b);
  const int q0 = tile * QUERIES + pair * 32, qi = q0 + c32;
  const bool there = qi < a.sq;
  const S *K = rows_of<EL>(a.k, b, hk), *V = rows_of<EL>(a.v, b, hk);
  const uint8_t *mask = reinterpret_cast<const uint8_t *>(a.mask.base) + (int64_t)b * a.mask.batch + (int64_t)h * a.mask.head;
  int seen = keys;
  if (a.causal) seen = min(seen, max(0, min((tile + 1) * QUERIES, a.sq) + a.shift));
  const int steps = (seen + KEYS - 1) / KEYS;

  const uint32_t lds = lds_address(stages);
  T kt, vt;
  kt.begin(wave, a.k.row);
  vt.begin(wave, a.v.row);
  if (a.dim != DP) {
    for (int s = 0; s < RING; s++) {
      kt.clear(lds + s * STAGE, a.dim);
      vt.clear(lds + s * STAGE + T::SIZE, a.dim);
    }
    __syncthreads();
  }
  const bool direct = a.k.direct && a.v.direct;
  auto fetch = [&](int t, uint32_t to) {  // tile by tile
    kt.fetch(K, keys - t * KEYS, a.k, a.dim, to);
    vt.fetch(V, keys - t * KEYS, a.v, a.dim, to + T::SIZE);
    K += KEYS * a.k.row;
    V += KEYS * a.v.row;
  };
  for (int t = 0; t < AHEAD && t < steps; t++) fetch(t, lds + t * STAGE);
  Column<EL, DP> q, g;
  g.load(rows_of<EL>(a.g, b, h) + (int64_t)qi * a.g.row, there, a.dim);
  q.load(rows_of<EL>(a.out, b, h) + (int64_t)qi * a.out.row, there, a.dim);
  float delta = g.dot(q);
  delta = delta + other_half(delta);
  q.load(rows_of<EL>(a.q, b, h) + (int64_t)qi * a.q.row, there, a.dim);
  float power = -INF;
  if (there) power = exponent_of<EL>(reinterpret_cast<const float *>(a.lse.base)[(int64_t)b * a.lse.batch + (int64_t)h * a.lse.head + (int64_t)qi * a.lse.row]);
  if (part == 0 && qi < a.rows_pitch) {  // for the second launch, 32 rows' powers and then their differences' starts; past the end -inf and 0
    float *to = a.rows + ((int64_t)bh * a.rows_pitch + q0) * 2;
    to[lane] = lane < 32 ? power : there ? -delta : 0.0f;
  }
  f32x16 dq[OT];
#pragma unroll
  for (int t = 0; t < OT; t++)
#pragma unroll
    for (int e = 0; e < 16; e++) dq[t][e] = 0.0f;
  Places<T, EL> places;
  places.begin();
  uint32_t stage = lds, ahead = lds + AHEAD * STAGE;
  for (int t = 0; t < steps; t++) {
    // this tile has come, and the stage that is filled next has been used
    if (AHEAD == 2 && t > 0 && (t + 2) * KEYS <= keys && t + 1 < steps && direct) meet<2 * T::LPW>();
    else meet<0>();
    if (t + AHEAD < steps) fetch(t + AHEAD, ahead);
    const uint32_t now = stage;
    stage = stage == lds + (RING - 1) * STAGE ? lds : stage + STAGE;
    ahead = ahead == lds + (RING - 1) * STAGE ? lds : ahead + STAGE;
    const int first = t * KEYS + part * 32;
    if (first >= keys || (a.causal && first > q0 + 31 + a.shift)) continue;  // nothing of it is seen
    const Places<T, EL> here = places.in(now + (uint32_t)(part * 32 * T::ROW));
    MaskBytes bytes;
    auto begin = [&](int r0, f32x16 &p, f32x16 &ds) {
      if constexpr (MASK) bytes.load_keys(a, mask, qi, first + r0);
#pragma unroll
      for (int e = 0; e < 16; e++) p[e] = 0.0f, ds[e] = -delta;
    };
    auto differences = [&](int r0, const f32x16 &p, f32x16 &ds) {
#pragma unroll
      for (int e = 0; e < 16; e++) ds[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[e], a.c2, power)) * ds[e];
      const int j0 = first + r0;
      if (!MASK && j0 + 32 <= keys && !(a.causal && j0 + 31 > q0 + a.shift)) return;
      uint32_t see = keys_seen(a, qi, j0, keys);
      if constexpr (MASK) see &= bytes.kept();
#pragma unroll
      for (int e = 0; e < 16; e++) ds[e] = (see >> e) & 1 ? ds[e] : 0.0f;
    };
    f32x16 p, ds;
    Weights<EL> w;
    RowElements<T, EL, OT> k;  // (on their way during the exponentials; those of heads of 128 would be more registers than there are)
    begin(0, p, ds);
    two_scores<T, 0>(p, q, ds, g, here, a.dim);
    if constexpr (DP <= 96) k.template load<0>(here);
    if constexpr (!EL::F32) in_order();
    differences(0, p, ds);
    if constexpr (DP > 96) k.template load<0>(here);
    w.set(ds);
    if constexpr (SUBS == 2) {
      k.add(dq, w);
      begin(32, p, ds);
      two_scores<T, 32 * T::ROW>(p, q, ds, g, here, a.dim);
      k.template load<32 * T::ROW>(here);
      in_order();
      differences(32, p, ds);
      w.set(ds);
    }
    k.add(dq, w);
  }
  if constexpr (KW == 2) {  // the odd wave of a pair hands over
    static_assert(sizeof(float) * 2 * OT * 16 * 64 <= sizeof(stages), "sums of two waves fit the stages");
    float(*over)[OT * 16][64] = reinterpret_cast<float(*)[OT * 16][64]>(stages);
    __syncthreads();
    if (part == 1) {
#pragma unroll
      for (int t = 0; t < OT; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) over[pair][t * 16 + e][lane] = dq[t][e];
    }
    __syncthreads();
    if (part == 1) return;
#pragma unroll
    for (int t = 0; t < OT; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) dq[t][e] = dq[t][e] + over[pair][t * 16 + e][lane];
  }
  if (there) store_column<EL, DP>(const_cast<S *>(rows_of<EL>(a.dq, b, h)) + (int64_t)qi * a.dq.row, dq, a.scale * UNLIFT<EL>, a.dim);
}

// Which of queries i0 + (e / 4) * 8 + g * 4 + e % 4 see key kj, the mask aside, bit e of the result.
__device__ __forceinline__ uint32_t queries_seeing(const AttentionArgs &a, int kj, int i0) {
  return a.causal ? rows_from(kj - a.shift - i0 - (int)((threadIdx.x >> 5) & 1) * 4) : 0xffffu;
}

// Where a block of the second launch is: its keys, and its part of what they are seen by, the query tiles of all heads that share
// them, one head after the other.
template <class EL, int QUERIES, int KEYS = 128>
struct KeysWalk {
  int b, hk, keys, first;  // batch, head, the sequence's keys, the block's first
  int part, steps;
  int tiles, before;  // a head's query tiles, and how many of them see none of the block's keys
  int at, head;       // tile and head of a step
  __device__ __forceinline__ KeysWalk(const AttentionArgs &a) {
    const uint32_t heads = (uint32_t)a.batch * (uint32_t)a.kv_heads, rest = blockIdx.x / heads;
    const int bh = (int)(blockIdx.x % heads), group = a.heads / a.kv_heads;
    b = bh / a.kv_heads;
    hk = bh % a.kv_heads;
    keys = keys_of(a, b);
    first = (int)(rest / (uint32_t)a.parts) * KEYS;  // the first keys first: under a causal mask most queries see them
    part = (int)(rest % (uint32_t)a.parts);
    tiles = (a.sq + QUERIES - 1) / QUERIES;
    before = a.causal ? min(tiles, max(0, first - a.shift) / QUERIES) : 0;
    const int64_t all = first < keys ? (int64_t)group * (tiles - before) : 0;
    const int64_t from = all * part / a.parts, to = all * (part + 1) / a.parts;
    steps = (int)(to - from);
    at = before, head = hk * group;
    if (steps > 0) {
      at += (int)(from % (tiles - before));
      head += (int)(from / (tiles - before));
    }
  }
  // Whether the next step is in another head.
  __device__ __forceinline__ bool next() {
    if (++at < tiles) return false;
    at = before;
    head++;
    return true;
  }
};

// A value of each of 32 rows, as the scores lie; `half`: the values' place, and 16 more in the wave's second half.
template <int OFFSET>
__device__ __forceinline__ void row_values(uint32_t half, f32x16 &x) {
#pragma unroll
  for (int e = 0; e < 16; e += 4) {
    const gemm_tile::f32x4 v = *at_lds<const lds_f32x4>(half + (uint32_t)(e * 8 + OFFSET));
#pragma unroll
    for (int j = 0; j < 4; j++) x[e + j] = v[j];
  }
}

// A column's sums: a key's dk or dv.
template <class EL, int DP, class W>
__device__ __forceinline__ void store_key(const AttentionArgs &a, const W &w, int kj, bool is_k, f32x16 (&acc)[DP / 32]) {
  if (kj >= w.keys) {  // a key that its sequence does not have saw zeros in its place: its gradients are zeros
#pragma unroll
    for (int t = 0; t < DP / 32; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[t][e] = 0.0f;
  }
  const float factor = is_k ? a.scale * UNLIFT<EL> : UNLIFT<EL>;
  if (a.partial) {
    float *to = a.partial + ((((int64_t)w.part * a.batch + w.b) * a.kv_heads + w.hk) * a.sk + kj) * 2 * a.dim;
    store_column<gemm_tile::ElF32, DP>(is_k ? to : to + a.dim, acc, factor, a.dim);
  } else {
    const HeadOperand &o = is_k ? a.dk : a.dv;
    store_column<EL, DP>(const_cast<typename EL::S *>(rows_of<EL>(o, w.b, w.hk)) + (int64_t)kj * o.row, acc, factor, a.dim);
  }
}

// For heads of up to 64. Blocks of four waves. KW = 1: each has 32 keys. KW = 2: two share 32 keys, each takes every other 32 queries of a
// tile, and their sums are added at the end: where there would be fewer than two blocks a unit ([4,12,1024,64] bfloat16 causal 32.7 and
// 30.8 us, [8,12,1024,64] 47 and 52; [2,12,1024,64] not causal 27.9 + 7.2 for sums of parts, and 27.4). What a block walks over is cut into
// a.parts, a block each, where there would still be few; their sums are joined by another launch.
template <class EL, int DP, int KW, bool MASK>
__global__ __launch_bounds__(256) void attention_grad_keys_kernel(AttentionArgs a) {
  constexpr int QUERIES = EL::F32 ? 32 : 64, OT = DP / 32;
  using T = Tile<EL, DP, QUERIES, 4>;
  constexpr int STAGE = 2 * T::SIZE + 1024, RING = 3, VALUES = 2 * T::SIZE;  // queries, their gradients, and each row's values
  __shared__ __attribute__((aligned(1024))) unsigned char stages[RING * STAGE];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pair = wave / KW, share = wave % KW;
  KeysWalk<EL, QUERIES, 128 / KW> w(a);
  const int k0 = w.first + pair * 32, kj = k0 + (threadIdx.x & 31);
  const uint32_t lds = lds_address(stages);
  T qt, gt;
  qt.begin(wave, a.q.row);
  gt.begin(wave, a.g.row);
  if (a.dim != DP) {
    for (int s = 0; s < RING; s++) {
      qt.clear(lds + s * STAGE, a.dim);
      gt.clear(lds + s * STAGE + T::SIZE, a.dim);
    }
    __syncthreads();
  }
  const bool direct = a.q.direct && a.g.direct;
  int at = w.at, head = w.head;  // of the step that is worked on (the walk's are of the one that is fetched)
  const typename EL::S *q_next, *g_next;
  const float *values_next;
  auto find = [&]() {  // the walk's place, where it is not behind the last one
    const int64_t i0 = (int64_t)w.at * QUERIES;
    q_next = rows_of<EL>(a.q, w.b, w.head) + i0 * a.q.row;
    g_next = rows_of<EL>(a.g, w.b, w.head) + i0 * a.g.row;
    values_next = a.rows + (((int64_t)w.b * a.heads + w.head) * a.rows_pitch + i0 + wave * 32) * 2;
  };
  // The walk's step, and on; whether all of it is on its way past the registers.
  auto fetch = [&](uint32_t to) {
    const int left = a.sq - w.at * QUERIES;
    qt.fetch(q_next, left, a.q, a.dim, to);
    gt.fetch(g_next, left, a.g, a.dim, to + T::SIZE);
    if (wave < QUERIES / 32) load_to_lds4(values_next, (threadIdx.x & 63) * 4, to + VALUES + wave * 256);
    q_next += QUERIES * a.q.row;
    g_next += QUERIES * a.g.row;
    values_next += QUERIES * 2;
    if (w.next()) find();
    return direct && left >= QUERIES;
  };
  if (w.steps > 0) find();
  bool whole = false;  // of the step after the one that is worked on
  if (w.steps > 0) fetch(lds);
  if (w.steps > 1) whole = fetch(lds + STAGE);
  Column<EL, DP> k, v;
  k.load(rows_of<EL>(a.k, w.b, w.hk) + (int64_t)kj * a.k.row, kj < w.keys, a.dim);
  v.load(rows_of<EL>(a.v, w.b, w.hk) + (int64_t)kj * a.v.row, kj < w.keys, a.dim);
  f32x16 dk[OT], dv[OT];
#pragma unroll
  for (int t = 0; t < OT; t++)
#pragma unroll
    for (int e = 0; e < 16; e++) dk[t][e] = dv[t][e] = 0.0f;
  Places<T, EL> places;
  places.begin();
  const uint32_t half16 = ((threadIdx.x >> 5) & 1) * 16;
  uint32_t stage = lds, ahead = lds + 2 * STAGE;
  for (int t = 0; t < w.steps; t++) {
    // this tile has come, and the stage that is filled next has been used
    if (t == 0 || !whole) meet<0>();
    else if (wave < QUERIES / 32) meet<2 * T::LPW + 1>();
    else meet<2 * T::LPW>();
    whole = false;
    if (t + 2 < w.steps) whole = fetch(ahead);
    const uint32_t now = stage;
    stage = stage == lds + 2 * STAGE ? lds : stage + STAGE;
    ahead = ahead == lds + 2 * STAGE ? lds : ahead + STAGE;
    const int i0 = at * QUERIES + share * 32, head_now = head;
    if (++at == w.tiles) at = w.before, head++;
    if (k0 >= w.keys || (a.causal && k0 > i0 + QUERIES / KW - 1 + a.shift)) continue;  // nothing of the tile sees these keys
    const Places<T, EL> here = places.in(now + (uint32_t)(share * 32 * T::ROW));
    uint32_t values = now + (uint32_t)share * 256 + half16;
    asm("" : "+v"(values));
    MaskBytes bytes;
    auto begin = [&](int r0, f32x16 &p) {
      if constexpr (MASK)
        bytes.load_queries(a, reinterpret_cast<const uint8_t *>(a.mask.base) + (int64_t)w.b * a.mask.batch + (int64_t)head_now * a.mask.head, kj, i0 + r0);
#pragma unroll
      for (int e = 0; e < 16; e++) p[e] = 0.0f;
    };
    auto differences = [&](int r0, const f32x16 &l, f32x16 &p, f32x16 &ds) {
#pragma unroll
      for (int e = 0; e < 16; e++) {
        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[e], a.c2, l[e]));
        ds[e] = p[e] * ds[e];
      }
      if (!MASK && !(a.causal && k0 + 31 > i0 + r0 + a.shift)) return;
      uint32_t seeing = queries_seeing(a, kj, i0 + r0);
      if constexpr (MASK) seeing &= bytes.kept();
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const bool keep = (seeing >> e) & 1;
        p[e] = keep ? p[e] : 0.0f;
        ds[e] = keep ? ds[e] : 0.0f;
      }
    };
    f32x16 p, ds, l;
    Weights<EL> pw, dsw;
    RowElements<T, EL, OT> g, q;  // (on their way during the exponentials)
    begin(0, p);
    row_values<VALUES + 128>(values, ds);
    two_scores<T, 0>(p, k, ds, v, here, a.dim);
    row_values<VALUES>(values, l);
    g.template load<T::SIZE>(here);
    q.template load<0>(here);
    if constexpr (!EL::F32) in_order();
    differences(0, l, p, ds);
    pw.set(p);
    dsw.set(ds);
    if constexpr (QUERIES / KW == 64) {
      g.add(dv, pw);
      q.add(dk, dsw);
      begin(32, p);
      row_values<VALUES + 256 + 128>(values, ds);
      two_scores<T, 32 * T::ROW>(p, k, ds, v, here, a.dim);
      row_values<VALUES + 256>(values, l);
      g.template load<T::SIZE + 32 * T::ROW>(here);
      q.template load<32 * T::ROW>(here);
      in_order();
      differences(32, l, p, ds);
      pw.set(p);
      dsw.set(ds);
    }
    g.add(dv, pw);
    q.add(dk, dsw);
  }
  if constexpr (KW == 2) {  // the odd wave of a pair hands over
    static_assert(sizeof(float) * 4 * OT * 16 * 64 <= sizeof(stages), "sums of two waves fit the stages");
    float(*over)[2 * OT * 16][64] = reinterpret_cast<float(*)[2 * OT * 16][64]>(stages);
    const int lane = threadIdx.x & 63;
    __syncthreads();
    if (share == 1) {
#pragma unroll
      for (int t = 0; t < OT; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) over[pair][t * 16 + e][lane] = dk[t][e], over[pair][(OT + t) * 16 + e][lane] = dv[t][e];
    }
    __syncthreads();
    if (share == 1) return;
#pragma unroll
    for (int t = 0; t < OT; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) dk[t][e] = dk[t][e] + over[pair][t * 16 + e][lane], dv[t][e] = dv[t][e] + over[pair][(OT + t) * 16 + e][lane];
  }
  if (kj >= a.sk) return;
  store_key<EL, DP>(a, w, kj, true, dk);
  store_key<EL, DP>(a, w, kj, false, dv);
}

// The same for heads of more than 64. Blocks of two pairs of waves (float32: four), of which the two of a pair have the same 32 keys: one
// makes the scores, p and dv, the other g . v, ds and dk, one tile of queries behind the first, whose p it takes from LDS. So a wave holds
// the vectors and the sums of one operand, not of two, which for heads of 128 are more registers than two waves of a unit's may have.
// Three stages: the tile that is on its way, and those of the two kinds of waves. (A fourth, for two tiles on their way, is 84 KB
// of 16-bit heads of 128: over half of a unit's LDS.)
template <class EL, int DP, int PAIRS, bool MASK>
__global__ __launch_bounds__(128 * PAIRS) __attribute__((amdgpu_waves_per_eu(2))) void attention_grad_wide_keys_kernel(AttentionArgs a) {
  constexpr int QUERIES = 32, OT = DP / 32;
  using T = Tile<EL, DP, QUERIES, PAIRS>;  // (half of the waves bring each operand's)
  constexpr int STAGE = 2 * T::SIZE + 1024, RING = 3, VALUES = 2 * T::SIZE;
  __shared__ __attribute__((aligned(1024))) unsigned char stages[RING * STAGE];
  __shared__ __attribute__((aligned(16))) float over[2][PAIRS][4][64][4];  // p, for the other wave: [tile][pair][e / 4][lane][e % 4]

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), pair = wave % PAIRS;
  const uint32_t lds = lds_address(stages);
  const uint32_t half16 = ((threadIdx.x >> 5) & 1) * 16;
  // The two kinds of waves have code of their own, which meets at the same barriers.
  auto run = [&](auto kind) {
    constexpr bool second = decltype(kind)::value;  // dk
    KeysWalk<EL, QUERIES, 32 * PAIRS> w(a);
    const int k0 = w.first + pair * 32, kj = k0 + (lane & 31);
    const HeadOperand &mine = second ? a.v : a.k, &brought = second ? a.g : a.q;
    T tile;
    tile.begin(pair, brought.row);
    if (a.dim != DP) {
      for (int s = 0; s < RING; s++) tile.clear(lds + s * STAGE + (second ? T::SIZE : 0), a.dim);
      meet<0>();
    }
    int at = w.at, head = w.head;  // of the step that this wave works on (the walk's are of the one that is fetched)
    const typename EL::S *next;
    const float *values_next;
    auto find = [&]() {  // the walk's place, where it is not behind the last one
      const int64_t i0 = (int64_t)w.at * QUERIES;
      next = rows_of<EL>(brought, w.b, w.head) + i0 * brought.row;
      values_next = a.rows + (((int64_t)w.b * a.heads + w.head) * a.rows_pitch + i0) * 2;
    };
    auto fetch = [&](uint32_t to) {
      const int left = a.sq - w.at * QUERIES;
      tile.fetch(next, left, brought, a.dim, to + (second ? T::SIZE : 0));
      if (!second && pair == 0) load_to_lds4(values_next, lane * 4, to + VALUES);
      next += QUERIES * brought.row;
      values_next += QUERIES * 2;
      if (w.next()) find();
    };
    if (w.steps > 0) {
      find();
      fetch(lds);
    }
    Column<EL, DP> own;
    own.load(rows_of<EL>(mine, w.b, w.hk) + (int64_t)kj * mine.row, kj < w.keys, a.dim);
    f32x16 acc[OT];
#pragma unroll
    for (int t = 0; t < OT; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[t][e] = 0.0f;
    Places<T, EL> places;
    places.begin();
    uint32_t stage = lds, ahead = lds + STAGE;
    for (int t = 0; w.steps > 0 && t <= w.steps; t++) {
      meet<0>();  // tile t has come, p of the tile before it too, and what is filled next has been used
      if (t + 1 < w.steps) fetch(ahead);
      ahead = ahead == lds + (RING - 1) * STAGE ? lds : ahead + STAGE;
      if (second ? t == 0 : t == w.steps) continue;
      const uint32_t now = stage;
      stage = stage == lds + (RING - 1) * STAGE ? lds : stage + STAGE;
      const int i0 = at * QUERIES, head_now = head;
      if (++at == w.tiles) at = w.before, head++;
      if (k0 >= w.keys || (a.causal && k0 > i0 + 31 + a.shift)) continue;  // nothing of the tile sees these keys
      float(*between)[64][4] = over[(second ? t - 1 : t) & 1][pair];
      const bool inner = !MASK && !(a.causal && k0 + 31 > i0 + a.shift);
      MaskBytes bytes;
      if constexpr (!second && MASK)
        bytes.load_queries(a, reinterpret_cast<const uint8_t *>(a.mask.base) + (int64_t)w.b * a.mask.batch + (int64_t)head_now * a.mask.head, kj, i0);
      const Places<T, EL> here = places.in(now);
      uint32_t values = now + half16;
      asm("" : "+v"(values));
      f32x16 x, l;  // l: the rows' powers; in the second wave p, which the first wave left
      if (second) {
        row_values<VALUES + 128>(values, x);
      } else {
#pragma unroll
        for (int e = 0; e < 16; e++) x[e] = 0.0f;
      }
      RowVectors<T, EL, DP> vectors;
      vectors.template load<(second ? T::SIZE : 0)>(here);
      if constexpr (!EL::F32) in_order();
      vectors.scores(x, own);
      if (second) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const gemm_tile::f32x4 p = *reinterpret_cast<const gemm_tile::f32x4 *>(between[e >> 2][lane]);
#pragma unroll
          for (int j = 0; j < 4; j++) l[e + j] = p[j];
        }
      } else {
        row_values<VALUES>(values, l);
      }
      RowElements<T, EL, OT> elements;  // (on their way during the exponentials)
      elements.template load<(second ? 0 : T::SIZE)>(here);
      if constexpr (!EL::F32) in_order();
      if (second) {
#pragma unroll
        for (int e = 0; e < 16; e++) x[e] = l[e] * x[e];
        if (!inner) {
#pragma unroll
          for (int e = 0; e < 16; e++) x[e] = l[e] != 0.0f ? x[e] : 0.0f;  // (what a query does not see may be no number)
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; e++) x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], a.c2, l[e]));
        if (!inner) {
          uint32_t seeing = queries_seeing(a, kj, i0);
          if constexpr (MASK) seeing &= bytes.kept();
#pragma unroll
          for (int e = 0; e < 16; e++) x[e] = (seeing >> e) & 1 ? x[e] : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 16; e += 4) *reinterpret_cast<gemm_tile::f32x4 *>(between[e >> 2][lane]) = gemm_tile::f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
      }
      Weights<EL> y;
      y.set(x);
      elements.add(acc, y);
    }
    if (kj < a.sk) store_key<EL, DP>(a, w, kj, second, acc);
  };
  if (wave >= PAIRS) run(std::integral_constant<bool, true>{});
  else run(std::integral_constant<bool, false>{});
}

// The parts' sums, in order, V elements of a row at a time. (There are parts for few rows only: all sizes fit 32 bits.)
template <class EL, int V>
__global__ __launch_bounds__(256) void attention_grad_join_kernel(AttentionArgs a) {
  using S = typename EL::S;
  const uint32_t of_row = 2u * (uint32_t)a.dim / V, rows = (uint32_t)a.batch * (uint32_t)a.kv_heads * (uint32_t)a.sk;
  const int64_t part = (int64_t)rows * 2 * a.dim;
  const uint32_t each = 256 / of_row, row = blockIdx.x * each + threadIdx.x / of_row;  // (a row has at most 256 elements)
  if (threadIdx.x >= each * of_row || row >= rows) return;
  const int at = (int)(threadIdx.x % of_row) * V;
  const float *from = a.partial + (int64_t)row * 2 * a.dim + at;
  float sum[V];
  __builtin_memcpy(sum, from, sizeof sum);
  for (int p = 1; p < a.parts; p++) {
    float more[V];
    __builtin_memcpy(more, from + p * part, sizeof more);
#pragma unroll
    for (int j = 0; j < V; j++) sum[j] = sum[j] + more[j];
  }
  const uint32_t bh = row / (uint32_t)a.sk, j = row - bh * (uint32_t)a.sk, b = bh / (uint32_t)a.kv_heads, h = bh - b * (uint32_t)a.kv_heads;
  const bool is_k = at < a.dim;
  const HeadOperand &o = is_k ? a.dk : a.dv;
  S *to = const_cast<S *>(rows_of<EL>(o, (int)b, (int)h)) + (int64_t)j * o.row + (is_k ? at : at - a.dim);
  if constexpr (EL::F32) {
    __builtin_memcpy(to, sum, sizeof sum);
  } else if constexpr (V == 4) {
    const uint32_t w[2] = {pack2<EL>(sum[0], sum[1]), pack2<EL>(sum[2], sum[3])};
    __builtin_memcpy(to, w, sizeof w);
  } else {
    *to = (uint16_t)pack2<EL>(sum[0], 0.0f);
  }
}

template <class EL, int DP, bool MASK>
void launch(nxh_context *ctx, AttentionArgs a, int keys_of_block) {
  const int units = ctx->compute_units > 0 ? ctx->compute_units : 256;
  const auto blocks_of = [&](int heads, int n) { return dim3((unsigned)(a.batch * heads * n)); };
  if (a.sq > 0 && a.heads > 0) {
    a.tiles = (a.sq + 127) / 128;
    if ((int64_t)a.batch * a.heads * a.tiles < 2 * units) {
      a.tiles = (a.sq + 63) / 64;
      hipLaunchKernelGGL((attention_grad_queries_kernel<EL, DP, 2, MASK>), blocks_of(a.heads, a.tiles), dim3(256), 0, ctx->stream, a);
    } else {
      hipLaunchKernelGGL((attention_grad_queries_kernel<EL, DP, 1, MASK>), blocks_of(a.heads, a.tiles), dim3(256), 0, ctx->stream, a);
    }
  }
  if (a.sk == 0) return;
  if constexpr (DP <= 64) {
    const dim3 grid = blocks_of(a.kv_heads, (a.sk + keys_of_block - 1) / keys_of_block * a.parts);
    if constexpr (!EL::F32) {
      if (keys_of_block == 64) hipLaunchKernelGGL((attention_grad_keys_kernel<EL, DP, 2, MASK>), grid, dim3(256), 0, ctx->stream, a);
    }
    if (keys_of_block == 128) hipLaunchKernelGGL((attention_grad_keys_kernel<EL, DP, 1, MASK>), grid, dim3(256), 0, ctx->stream, a);
  } else {
    constexpr int PAIRS = EL::F32 ? 4 : 2;
    hipLaunchKernelGGL((attention_grad_wide_keys_kernel<EL, DP, PAIRS, MASK>), blocks_of(a.kv_heads, (a.sk + 32 * PAIRS - 1) / (32 * PAIRS) * a.parts),
                       dim3(128 * PAIRS), 0, ctx->stream, a);
  }
  if (!a.partial) return;
  const int v = a.dim % 4 == 0 ? 4 : 1, each = 256 / (2 * a.dim / v), rows = a.batch * a.kv_heads * a.sk;
  const dim3 grid((unsigned)((rows + (int64_t)each - 1) / each));
  if (v == 4) hipLaunchKernelGGL((attention_grad_join_kernel<EL, 4>), grid, dim3(256), 0, ctx->stream, a);
  else hipLaunchKernelGGL((attention_grad_join_kernel<EL, 1>), grid, dim3(256), 0, ctx->stream, a);
}
template <class EL, int DP>
void launch_mask(nxh_context *ctx, const AttentionArgs &a, int keys_of_block) {
  if (a.mask.base) launch<EL, DP, true>(ctx, a, keys_of_block);
  else launch<EL, DP, false>(ctx, a, keys_of_block);
}
template <class EL>
void launch_dim(nxh_context *ctx, const AttentionArgs &a, int keys_of_block) {
  if (a.dim <= 32) launch_mask<EL, 32>(ctx, a, keys_of_block);
  else if (a.dim <= 64) launch_mask<EL, 64>(ctx, a, keys_of_block);
  else if (a.dim <= 96) launch_mask<EL, 96>(ctx, a, keys_of_block);
  else launch_mask<EL, 128>(ctx, a, keys_of_block);
}

}  // namespace

NXH_EXPORT int nxh_attention_grad(nxh_context *ctx, const nxh_tensor *dq, const nxh_tensor *dk, const nxh_tensor *dv, const nxh_tensor *g,
                                  const nxh_tensor *q, const nxh_tensor *k, const nxh_tensor *v, const nxh_tensor *out, const nxh_tensor *lse,
                                  const nxh_tensor *lengths, const nxh_tensor *mask, double scale, int causal) {
  NXH_DEFER_TOUCH(ctx, 3, dq, dk, dv, g, q, k, v, out, lse, lengths, mask);
  const char *op = "attention_grad";
  if (!ctx || !dq || !dk || !dv || !g || !q || !k || !v || !out || !lse) return nxh_fail(NXH_INVALID_ARGUMENT, op, "null argument");
  int rc;
  for (const nxh_tensor *t : {dq, dk, dv, g, q, k, v, out, lse, lengths, mask})
    if (t && (rc = nxh_check_tensor(op, t))) return rc;
  AttentionArgs a;
  if ((rc = attention_arguments(op, a, q, k, v, out, lse, lengths, mask, scale, causal, true))) return rc;
  const int dt = q->dtype;
  if ((rc = attention_operand(op, g, dt, a.batch, a.heads, a.sq, a.dim, a.g, false)) || (rc = attention_operand(op, dq, dt, a.batch, a.heads, a.sq, a.dim, a.dq, true)) ||
      (rc = attention_operand(op, dk, dt, a.batch, a.kv_heads, a.sk, a.dim, a.dk, true)) || (rc = attention_operand(op, dv, dt, a.batch, a.kv_heads, a.sk, a.dim, a.dv, true)))
    return rc;
  if (a.batch == 0 || a.kv_heads == 0) return NXH_OK;
  const nxh_tensor *results[] = {dq, dk, dv}, *inputs[] = {g, q, k, v, out, lse, lengths, mask};
  for (const nxh_tensor *r : results)
    for (const nxh_tensor *i : inputs)
      if (i && same_start(r, i)) return nxh_fail(NXH_INVALID_ARGUMENT, op, "a gradient must not replace an input");
  if (same_start(dq, dk) || same_start(dq, dv) || same_start(dk, dv)) return nxh_fail(NXH_INVALID_ARGUMENT, op, "two gradients in one place");
  // A block has the keys that four waves or pairs of waves have and walks over all queries that see them: cut into parts where
  // that leaves units without work, down to parts of four tiles. A unit has room for one block of float32 heads of more than 64,
  // else for two. Under a causal mask the first blocks walk over twice the mean: wide heads take twice as many parts, and the last
  // ones fill the gaps ([1,16,8192,128] 757 us, and 697 + 15 for the sums).
  const int units = ctx->compute_units > 0 ? ctx->compute_units : 256;
  const bool wide = a.dim > 64, f32 = dt == NXH_F32;
  const int64_t heads = (int64_t)a.batch * a.kv_heads;
  const int keys_of_block = !f32 && (wide || heads * ((a.sk + 127) / 128) < 2 * units) ? 64 : 128;
  const int64_t blocks = heads * ((a.sk + keys_of_block - 1) / keys_of_block), walk = (int64_t)(a.heads / a.kv_heads) * ((a.sq + 31) / 32);
  const int64_t room = (wide ? (f32 ? 1 : 2) * (a.causal ? 2 : 1) : 2) * (int64_t)units;
  a.parts = blocks > 0 && walk > 0 ? (int)std::max<int64_t>(1, std::min<int64_t>({16, room / blocks, walk / 4})) : 1;
  if ((double)blocks * a.parts > 2147483647.0) return nxh_fail(NXH_FAILURE, op, "too many rows for one launch");
  std::lock_guard<std::mutex> guard(ctx->mu);
  NXH_HIP(op, hipSetDevice(ctx->device));
  a.rows_pitch = (a.sq + 63) / 64 * 64;
  const size_t rows = (size_t)a.batch * a.heads * a.rows_pitch * 8;
  const size_t sums = a.parts > 1 ? (size_t)a.parts * a.batch * a.kv_heads * a.sk * 2 * a.dim * 4 : 0;
  void *space = nullptr;
  if ((rc = nxh_alloc_locked(ctx, rows + sums, &space))) return rc;
  a.rows = (float *)space;
  a.partial = sums ? (float *)((char *)space + rows) : nullptr;
  nxh_set_path("attention_grad");
  if (dt == NXH_F32) launch_dim<gemm_tile::ElF32>(ctx, a, keys_of_block);
  else if (dt == NXH_BF16) launch_dim<gemm_tile::ElBF16>(ctx, a, keys_of_block);
  else launch_dim<gemm_tile::ElF16>(ctx, a, keys_of_block);
  nxh_free_locked(ctx, space);  // (the stream orders its next use behind these launches)
  NXH_HIP(op, hipGetLastError());
  return NXH_OK;
}
