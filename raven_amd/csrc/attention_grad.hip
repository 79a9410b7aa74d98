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

// Blocks of four waves with 32 queries each.
template <class EL, int DP>
__global__ __launch_bounds__(256) void attention_grad_queries_kernel(AttentionArgs a) {
  using S = typename EL::S;
  constexpr int KEYS = EL::F32 ? 32 : 64, QUERIES = 128, OT = DP / 32;
  using T = Tile<EL, DP, KEYS>;
  constexpr int STAGE = 2 * T::SIZE;
  __shared__ __attribute__((aligned(16))) S stages[2 * STAGE];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c32 = lane & 31;
  const uint32_t heads = (uint32_t)a.batch * (uint32_t)a.heads;
  const int tile = a.tiles - 1 - (int)(blockIdx.x / heads);
  const int bh = (int)(blockIdx.x % heads), b = bh / a.heads, h = bh % a.heads, hk = h / (a.heads / a.kv_heads);
  const int keys = keys_of(a, b);
  const int q0 = tile * QUERIES + wave * 32, qi = q0 + c32;
  const bool there = qi < a.sq;
  const S *K = rows_of<EL>(a.k, b, hk), *V = rows_of<EL>(a.v, b, hk);
  const uint8_t *mask = a.mask.base ? reinterpret_cast<const uint8_t *>(a.mask.base) + (int64_t)b * a.mask.batch + (int64_t)h * a.mask.head : nullptr;
  int seen = keys;
  if (a.causal) seen = min(seen, max(0, min((tile + 1) * QUERIES, a.sq) + a.shift));
  const int steps = (seen + KEYS - 1) / KEYS;

  T kt, vt;
  kt.begin(a.k.row);
  vt.begin(a.v.row);
  auto fetch = [&](int t) {
    kt.fetch(K, a.k.row, t * KEYS, keys, a.dim);
    vt.fetch(V, a.v.row, t * KEYS, keys, a.dim);
  };
  auto lay = [&](int t) {
    kt.lay(stages + (t & 1) * STAGE);
    vt.lay(stages + (t & 1) * STAGE + T::SIZE);
  };
  if (steps > 0) {
    fetch(0);
    lay(0);
    if (steps > 1) fetch(1);
  }
  Column<EL, DP> q, g;
  g.load(rows_of<EL>(a.g, b, h) + (int64_t)qi * a.g.row, there, a.dim);
  q.load(rows_of<EL>(a.out, b, h) + (int64_t)qi * a.out.row, there, a.dim);
  float delta = g.dot(q);
  delta = delta + other_half(delta);
  q.load(rows_of<EL>(a.q, b, h) + (int64_t)qi * a.q.row, there, a.dim);
  float power = -INF;
  if (there) {
    power = exponent_of<EL>(reinterpret_cast<const float *>(a.lse.base)[(int64_t)b * a.lse.batch + (int64_t)h * a.lse.head + (int64_t)qi * a.lse.row]);
    if (lane < 32) a.delta[(int64_t)bh * a.sq + qi] = delta;
  }
  f32x16 dq[OT];
#pragma unroll
  for (int t = 0; t < OT; t++)
#pragma unroll
    for (int e = 0; e < 16; e++) dq[t][e] = 0.0f;
  for (int t = 0; t < steps; t++) {
    __syncthreads();  // this tile is there, and the one before has been used
    if (t + 1 < steps) {
      lay(t + 1);
      if (t + 2 < steps) fetch(t + 2);
    }
    const S *stage = stages + (t & 1) * STAGE;
#pragma unroll
    for (int sub = 0; sub < KEYS / 32; sub++) {
      const int r0 = sub * 32, j0 = t * KEYS + r0;
      if (j0 >= keys || (a.causal && j0 > q0 + 31 + a.shift)) continue;  // nothing of it is seen
      f32x16 p, ds;
#pragma unroll
      for (int e = 0; e < 16; e++) p[e] = 0.0f, ds[e] = -delta;
      rows_by_columns<EL, DP, T::PITCH>(p, stage + r0 * T::PITCH, q);
      rows_by_columns<EL, DP, T::PITCH>(ds, stage + T::SIZE + r0 * T::PITCH, g);
#pragma unroll
      for (int e = 0; e < 16; e++) ds[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[e], a.c2, power)) * ds[e];
      if (mask || j0 + 32 > keys || (a.causal && j0 + 31 > q0 + a.shift)) {
        const uint32_t see = keys_seen(a, mask, qi, j0, keys);
#pragma unroll
        for (int e = 0; e < 16; e++) ds[e] = (see >> e) & 1 ? ds[e] : 0.0f;
      }
      Weights<EL> w;
      w.set(ds);
      add_weighted_rows<EL, DP, T::PITCH>(dq, stage + r0 * T::PITCH, w);
    }
  }
  if (there) store_column<EL, DP>(const_cast<S *>(rows_of<EL>(a.dq, b, h)) + (int64_t)qi * a.dq.row, dq, a.scale * UNLIFT<EL>, a.dim);
}

// Which of queries i0 + (e / 4) * 8 + g * 4 + e % 4 see key kj, bit e of the result.
__device__ __forceinline__ uint32_t queries_seeing(const AttentionArgs &a, const uint8_t *mask, int kj, int i0) {
  const int g = (threadIdx.x >> 5) & 1, first = i0 + g * 4, from = a.causal ? kj - a.shift - first : 0;
  uint32_t seeing = 0;
#pragma unroll
  for (int e = 0; e < 16; e++) seeing |= (uint32_t)(!a.causal || (e >> 2) * 8 + (e & 3) >= from) << e;
  if (!mask) return seeing;
  const uint8_t *m = mask + (int64_t)(kj < a.sk ? kj : a.sk - 1) * a.mask_col;
  uint32_t kept = 0;
#pragma unroll
  for (int e = 0; e < 16; e++) {
    const int i = first + (e >> 2) * 8 + (e & 3);
    kept |= (uint32_t)(m[(int64_t)(i < a.sq ? i : a.sq - 1) * a.mask.row] != 0) << e;
  }
  return seeing & kept;
}

// Blocks of four waves with 32 keys each. What a block walks over, the query tiles of all heads that share its keys, is cut into
// a.parts, a block each, where there would be few blocks; their sums are joined by another launch.
template <class EL, int DP>
__global__ __launch_bounds__(256) void attention_grad_keys_kernel(AttentionArgs a) {
  using S = typename EL::S;
  constexpr int QUERIES = EL::F32 || DP > 96 ? 32 : 64, KEYS = 128, OT = DP / 32;
  using T = Tile<EL, DP, QUERIES>;
  constexpr int STAGE = 2 * T::SIZE;
  __shared__ __attribute__((aligned(16))) S stages[2 * STAGE];
  __shared__ __attribute__((aligned(16))) float powers[2][QUERIES], deltas[2][QUERIES];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c32 = lane & 31, half = lane >> 5;
  const uint32_t heads = (uint32_t)a.batch * (uint32_t)a.kv_heads;
  const uint32_t rest = blockIdx.x / heads;
  const int tile = (int)(rest / (uint32_t)a.parts), part = (int)(rest % (uint32_t)a.parts);  // the first keys first: under a causal mask most see them
  const int bh = (int)(blockIdx.x % heads), b = bh / a.kv_heads, hk = bh % a.kv_heads, group = a.heads / a.kv_heads;
  const int keys = keys_of(a, b);
  const int k0 = tile * KEYS + wave * 32, kj = k0 + c32;
  const bool there = kj < a.sk;
  Column<EL, DP> k, v;
  k.load(rows_of<EL>(a.k, b, hk) + (int64_t)kj * a.k.row, kj < keys, a.dim);
  v.load(rows_of<EL>(a.v, b, hk) + (int64_t)kj * a.v.row, kj < keys, a.dim);

  const int tiles = (a.sq + QUERIES - 1) / QUERIES;
  const int before = a.causal ? min(tiles, max(0, tile * KEYS - a.shift) / QUERIES) : 0;  // tiles whose queries see none of the block's keys
  const int64_t all = tile * KEYS < keys ? (int64_t)group * (tiles - before) : 0;
  const int64_t from = all * part / a.parts, to = all * (part + 1) / a.parts;
  const int steps = (int)(to - from);
  // where the walk is: query tile and head of the step that is fetched next
  int at = steps > 0 ? before + (int)(from % (tiles - before)) : 0, head = hk * group + (steps > 0 ? (int)(from / (tiles - before)) : 0);

  T qt, gt;
  qt.begin(a.q.row);
  gt.begin(a.g.row);
  float power = -INF, delta = 0.0f;
  int i0_now = 0, head_now = 0, i0_next = 0, head_next = 0;  // of the tile that is worked on, and of the one that was fetched last
  auto fetch = [&]() {
    const int i0 = at * QUERIES;
    qt.fetch(rows_of<EL>(a.q, b, head), a.q.row, i0, a.sq, a.dim);
    gt.fetch(rows_of<EL>(a.g, b, head), a.g.row, i0, a.sq, a.dim);
    if (threadIdx.x < QUERIES) {
      const int i = i0 + threadIdx.x;
      power = -INF, delta = 0.0f;
      if (i < a.sq) {
        power = reinterpret_cast<const float *>(a.lse.base)[(int64_t)b * a.lse.batch + (int64_t)head * a.lse.head + (int64_t)i * a.lse.row];
        delta = a.delta[((int64_t)b * a.heads + head) * a.sq + i];
      }
    }
    i0_next = i0, head_next = head;
    if (++at == tiles) at = before, head++;
  };
  auto lay = [&](int t) {
    qt.lay(stages + (t & 1) * STAGE);
    gt.lay(stages + (t & 1) * STAGE + T::SIZE);
    if (threadIdx.x < QUERIES) {
      powers[t & 1][threadIdx.x] = exponent_of<EL>(power);
      deltas[t & 1][threadIdx.x] = -delta;
    }
  };
  f32x16 dk[OT], dv[OT];
#pragma unroll
  for (int t = 0; t < OT; t++)
#pragma unroll
    for (int e = 0; e < 16; e++) dk[t][e] = dv[t][e] = 0.0f;
  if (steps > 0) {
    fetch();
    i0_now = i0_next, head_now = head_next;
    lay(0);
    if (steps > 1) fetch();
  }
  for (int t = 0; t < steps; t++) {
    __syncthreads();  // this tile is there, and the one before has been used
    const int i0_t = i0_now, head_t = head_now;
    if (t + 1 < steps) {
      lay(t + 1);
      i0_now = i0_next, head_now = head_next;
      if (t + 2 < steps) fetch();
    }
    const S *stage = stages + (t & 1) * STAGE;
    const uint8_t *mask = a.mask.base ? reinterpret_cast<const uint8_t *>(a.mask.base) + (int64_t)b * a.mask.batch + (int64_t)head_t * a.mask.head : nullptr;
#pragma unroll
    for (int sub = 0; sub < QUERIES / 32; sub++) {
      const int r0 = sub * 32, i0 = i0_t + r0;
      if (i0 >= a.sq || k0 >= keys || (a.causal && k0 > i0 + 31 + a.shift)) continue;  // nothing of it sees these keys
      f32x16 p, ds;
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const gemm_tile::f32x4 d = *reinterpret_cast<const gemm_tile::f32x4 *>(&deltas[t & 1][r0 + e * 2 + half * 4]);
#pragma unroll
        for (int j = 0; j < 4; j++) p[e + j] = 0.0f, ds[e + j] = d[j];
      }
      rows_by_columns<EL, DP, T::PITCH>(p, stage + r0 * T::PITCH, k);
      rows_by_columns<EL, DP, T::PITCH>(ds, stage + T::SIZE + r0 * T::PITCH, v);
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const gemm_tile::f32x4 w = *reinterpret_cast<const gemm_tile::f32x4 *>(&powers[t & 1][r0 + e * 2 + half * 4]);
#pragma unroll
        for (int j = 0; j < 4; j++) p[e + j] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[e + j], a.c2, w[j]));
      }
#pragma unroll
      for (int e = 0; e < 16; e++) ds[e] = p[e] * ds[e];
      if (mask || (a.causal && k0 + 31 > i0 + a.shift)) {
        const uint32_t seeing = queries_seeing(a, mask, kj, i0);
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const bool keep = (seeing >> e) & 1;
          p[e] = keep ? p[e] : 0.0f;
          ds[e] = keep ? ds[e] : 0.0f;
        }
      }
      Weights<EL> w;
      w.set(p);
      add_weighted_rows<EL, DP, T::PITCH>(dv, stage + T::SIZE + r0 * T::PITCH, w);
      w.set(ds);
      add_weighted_rows<EL, DP, T::PITCH>(dk, stage + r0 * T::PITCH, w);
    }
  }
  if (!there) return;
  // a key that its sequence does not have saw zeros in its place: its gradients are zeros
  const float one = kj < keys ? UNLIFT<EL> : 0.0f;
  if (kj >= keys) {
#pragma unroll
    for (int t = 0; t < OT; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) dk[t][e] = dv[t][e] = 0.0f;
  }
  if (a.partial) {
    float *to_k = a.partial + ((((int64_t)part * a.batch + b) * a.kv_heads + hk) * a.sk + kj) * 2 * a.dim;
    store_column<gemm_tile::ElF32, DP>(to_k, dk, a.scale * one, a.dim);
    store_column<gemm_tile::ElF32, DP>(to_k + a.dim, dv, one, a.dim);
  } else {
    store_column<EL, DP>(const_cast<S *>(rows_of<EL>(a.dk, b, hk)) + (int64_t)kj * a.dk.row, dk, a.scale * one, a.dim);
    store_column<EL, DP>(const_cast<S *>(rows_of<EL>(a.dv, b, hk)) + (int64_t)kj * a.dv.row, dv, one, a.dim);
  }
}

// The parts' sums, in order.
template <class EL>
__global__ __launch_bounds__(256) void attention_grad_join_kernel(AttentionArgs a) {
  using S = typename EL::S;
  const int64_t row = 2 * (int64_t)a.dim, size = (int64_t)a.batch * a.kv_heads * a.sk * row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < size; i += (int64_t)gridDim.x * 256) {
    float sum = a.partial[i];
    for (int p = 1; p < a.parts; p++) sum = sum + a.partial[(int64_t)p * size + i];
    const int64_t r = i / row;
    const int at = (int)(i - r * row), j = (int)(r % a.sk), bh = (int)(r / a.sk), b = bh / a.kv_heads, h = bh % a.kv_heads;
    const bool is_k = at < a.dim;
    const HeadOperand &o = is_k ? a.dk : a.dv;
    S *to = const_cast<S *>(rows_of<EL>(o, b, h)) + (int64_t)j * o.row + (is_k ? at : at - a.dim);
    if constexpr (EL::F32) *to = sum;
    else *to = (uint16_t)pack2<EL>(sum, 0.0f);
  }
}

template <class EL, int DP>
void launch(nxh_context *ctx, AttentionArgs a) {
  if (a.sq > 0 && a.heads > 0) {
    a.tiles = (a.sq + 127) / 128;
    hipLaunchKernelGGL((attention_grad_queries_kernel<EL, DP>), dim3((unsigned)(a.batch * a.heads * a.tiles)), dim3(256), 0, ctx->stream, a);
  }
  if (a.sk == 0) return;
  a.tiles = (a.sk + 127) / 128;
  hipLaunchKernelGGL((attention_grad_keys_kernel<EL, DP>), dim3((unsigned)(a.batch * a.kv_heads * a.tiles * a.parts)), dim3(256), 0, ctx->stream, a);
  if (!a.partial) return;
  const int64_t size = (int64_t)a.batch * a.kv_heads * a.sk * 2 * a.dim;
  hipLaunchKernelGGL((attention_grad_join_kernel<EL>), dim3((unsigned)std::min<int64_t>((size + 255) / 256, 1 << 16)), dim3(256), 0, ctx->stream, a);
}
template <class EL>
void launch_dim(nxh_context *ctx, const AttentionArgs &a) {
  if (a.dim <= 32) launch<EL, 32>(ctx, a);
  else if (a.dim <= 64) launch<EL, 64>(ctx, a);
  else if (a.dim <= 96) launch<EL, 96>(ctx, a);
  else launch<EL, 128>(ctx, a);
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
  const nxh_tensor *results[] = {dq, dk, dv}, *inputs[] = {g, q, k, v, out};
  for (const nxh_tensor *r : results)
    for (const nxh_tensor *i : inputs)
      if (same_start(r, i)) return nxh_fail(NXH_INVALID_ARGUMENT, op, "a gradient must not replace an input");
  // A block has 128 keys of a head and walks over all queries that see them: cut into parts where that leaves units
  // without work, down to parts of two tiles.
  const int units = ctx->compute_units > 0 ? ctx->compute_units : 256;
  const int64_t blocks = (int64_t)a.batch * a.kv_heads * ((a.sk + 127) / 128), walk = (int64_t)(a.heads / a.kv_heads) * ((a.sq + 63) / 64);
  a.parts = blocks > 0 && walk > 0 ? (int)std::max<int64_t>(1, std::min<int64_t>({16, 2 * units / blocks, walk / 2})) : 1;
  if ((double)blocks * a.parts > 2147483647.0) return nxh_fail(NXH_FAILURE, op, "too many rows for one launch");
  std::lock_guard<std::mutex> guard(ctx->mu);
  NXH_HIP(op, hipSetDevice(ctx->device));
  const size_t rows = ((size_t)a.batch * a.heads * a.sq * 4 + 255) / 256 * 256;
  const size_t sums = a.parts > 1 ? (size_t)a.parts * a.batch * a.kv_heads * a.sk * 2 * a.dim * 4 : 0;
  void *space = nullptr;
  if ((rc = nxh_alloc_locked(ctx, rows + sums, &space))) return rc;
  a.delta = (float *)space;
  a.partial = sums ? (float *)((char *)space + rows) : nullptr;
  nxh_set_path("attention_grad");
  if (dt == NXH_F32) launch_dim<gemm_tile::ElF32>(ctx, a);
  else if (dt == NXH_BF16) launch_dim<gemm_tile::ElBF16>(ctx, a);
  else launch_dim<gemm_tile::ElF16>(ctx, a);
  nxh_free_locked(ctx, space);  // (the stream orders its next use behind these launches)
  NXH_HIP(op, hipGetLastError());
  return NXH_OK;
}
