// attention_train.hip — nxh_attention_train: attention whose gradient follows. For a query i and the keys j it
// sees (below its sequence's length, j <= i + keys - queries where causal, and where the mask has it)
//   s_j = scale q . k_j,  lse = log sum e^(s_j),  out = sum e^(s_j - lse) v_j
// A query that sees none has out 0 and lse -inf. lse is what attention_grad.hip makes the probabilities from again.
//
// One pass over the keys. Scores stay unscaled, e^(scale (s - m)) = 2^(c s - c m), c = scale log2(e): one fused
// step and one power each. The reference m follows the largest score only once that is 2^8 above it, so that most
// tiles scale no results; what an exponential has too much, its sum has too. Sums, lse and results are float32; an
// exponential is rounded to 16 bits for the product with v, which then is the instruction's own (float32 operands: as it is).
//
// A lane has a query: scores come transposed (K Q^T), so its maximum and sum need one exchange between the wave's halves, and as they
// lie they are the second product's operand, of whose 32 keys an instruction takes those that one half of the wave holds.
// Tiles of keys go to LDS past the registers, two on their way where three stages fit half of a unit's LDS, else one (Tile, Places).
//
// What bounds it: of heads of 128 the matrix instructions and the vector unit by turns ([1,16,8192,128] bfloat16 causal 305 to 314 us, 875 to 901
// TFLOP/s; a product of 8192^3 reaches 1259 here); of heads of 64, whose 32 x 32 scores take 256 cycles of products and about 560 of
// exponentials, sums and rounding, the vector unit and each block's walk from tile to tile ([8,12,1024,64] 27 to 28 us).

#include "attention_tiles.hpp"

namespace {

// Blocks of four waves. KW = 1: each has 32 queries of 128. KW = 2: two share 32 queries, each takes every other 32 keys
// of a tile, and their results are joined at the end: twice the blocks.
template <class EL, int DP, int KW, bool MASK>
__global__ __launch_bounds__(256) void attention_train_kernel(AttentionArgs a) {
  using S = typename EL::S;
  constexpr int KEYS = !EL::F32 && DP <= 64 ? 64 : 32 * KW, SUBS = KEYS / 32 / KW, QUERIES = 128 / KW, OT = DP / 32;
  using T = Tile<EL, DP, KEYS, 4>;
  constexpr int STAGE = 2 * T::SIZE, RING = 3 * STAGE <= 80 * 1024 ? 3 : 2, AHEAD = RING - 1;  // tiles on their way
  __shared__ __attribute__((aligned(1024))) unsigned char stages[RING * STAGE];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c32 = lane & 31;
  const int pair = wave / KW, part = wave % KW;
  const uint32_t heads = (uint32_t)a.batch * (uint32_t)a.heads;
  const int tile = a.tiles - 1 - (int)(blockIdx.x / heads);  // the last queries first: under a causal mask they see most
  const int bh = (int)(blockIdx.x % heads), b = bh / a.heads, h = bh % a.heads, hk = h / (a.heads / a.kv_heads);
  const int keys = keys_of(a, b);
  const int q0 = tile * QUERIES + pair * 32, qi = q0 + c32;
  const S *K = rows_of<EL>(a.k, b, hk), *V = rows_of<EL>(a.v, b, hk);
  const uint8_t *mask = reinterpret_cast<const uint8_t *>(a.mask.base) + (int64_t)b * a.mask.batch + (int64_t)h * a.mask.head;

  int seen = keys;  // by the block's last query
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
  Column<EL, DP> q;
  q.load(rows_of<EL>(a.q, b, h) + (int64_t)qi * a.q.row, qi < a.sq, a.dim);

  f32x16 out[OT];
#pragma unroll
  for (int t = 0; t < OT; t++)
#pragma unroll
    for (int e = 0; e < 16; e++) out[t][e] = 0.0f;
  float m = -INF, sum = 0.0f;
  float mc = 0.0f, lim = INF;  // -c m, and +inf before the first score, where exponentials take 0
  Places<T, EL> places;
  places.begin();
  uint32_t stage = lds, ahead = lds + AHEAD * STAGE;
  for (int t = 0; t < steps; t++) {
    // this tile has come, and the stage that is filled next has been used
    if (AHEAD == 2 && t > 0 && t + 1 < steps && (t + 2) * KEYS <= keys && direct) meet<2 * T::LPW>();
    else meet<0>();
    if (t + AHEAD < steps) fetch(t + AHEAD, ahead);
    const Places<T, EL> here = places.in(stage + (uint32_t)(part * 32 * T::ROW));
    stage = stage == lds + (RING - 1) * STAGE ? lds : stage + STAGE;
    ahead = ahead == lds + (RING - 1) * STAGE ? lds : ahead + STAGE;
    const int j0 = t * KEYS + part * 32;
    if (j0 >= keys || (a.causal && j0 > q0 + 31 + a.shift)) continue;  // nothing of it is seen
    MaskBytes bytes[SUBS];
    if constexpr (MASK) {
#pragma unroll
      for (int u = 0; u < SUBS; u++) bytes[u].load_keys(a, mask, qi, j0 + u * 32);
    }
    f32x16 s[SUBS];
    RowVectors<T, EL, DP> k[SUBS];
    k[0].template load<0>(here);
    if constexpr (SUBS == 2) k[1].template load<32 * T::ROW>(here);
    if constexpr (!EL::F32) in_order();
#pragma unroll
    for (int u = 0; u < SUBS; u++) {
#pragma unroll
      for (int e = 0; e < 16; e++) s[u][e] = 0.0f;
      k[u].scores(s[u], q);
    }
    RowElements<T, EL, OT> v[SUBS];  // (on their way during the exponentials)
    v[0].template load<T::SIZE>(here);
    if constexpr (SUBS == 2) v[1].template load<T::SIZE + 32 * T::ROW>(here);
    if constexpr (!EL::F32) in_order();
    if (MASK || j0 + SUBS * 32 > keys || (a.causal && j0 + SUBS * 32 - 1 > q0 + a.shift)) {
#pragma unroll
      for (int u = 0; u < SUBS; u++) {
        uint32_t see = keys_seen(a, qi, j0 + u * 32, keys);
        if constexpr (MASK) see &= bytes[u].kept();
#pragma unroll
        for (int e = 0; e < 16; e++) s[u][e] = (see >> e) & 1 ? s[u][e] : -INF;
      }
    }
    float most = s[0][0];
#pragma unroll
    for (int u = 0; u < SUBS; u++)
#pragma unroll
      for (int e = 0; e < 16; e++) most = __builtin_fmaxf(most, s[u][e]);
    most = __builtin_fmaxf(most, other_half(most));
    const bool grow = most > m && __builtin_fmaf(most, a.c2, lim) > 8.0f;
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
      const float mc_new = -most * a.c2;
      const float alpha = grow ? __builtin_amdgcn_exp2f(__builtin_fmaf(m, a.c2, mc_new)) : 1.0f;
      m = grow ? most : m;
      mc = grow ? mc_new : mc;
      lim = grow ? mc_new : lim;
      sum = sum * alpha;
#pragma unroll
      for (int o = 0; o < OT; o++)
#pragma unroll
        for (int e = 0; e < 16; e++) out[o][e] = out[o][e] * alpha;
    }
#pragma unroll
    for (int u = 0; u < SUBS; u++) {
      float add = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; e++) {
        s[u][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][e], a.c2, mc));
        add = add + s[u][e];
      }
      sum = sum + add;
      Weights<EL> p;
      p.set(s[u]);
      v[u].add(out, p);
    }
  }
  if constexpr (KW == 2) {  // the odd wave of a pair hands over
    static_assert(sizeof(float) * 2 * (OT * 16 + 2) * 64 <= sizeof(stages), "results of two waves fit the stages");
    float(*over)[OT * 16 + 2][64] = reinterpret_cast<float(*)[OT * 16 + 2][64]>(stages);
    __syncthreads();
    if (part == 1) {
#pragma unroll
      for (int o = 0; o < OT; o++)
#pragma unroll
        for (int e = 0; e < 16; e++) over[pair][o * 16 + e][lane] = out[o][e];
      over[pair][OT * 16][lane] = m;
      over[pair][OT * 16 + 1][lane] = sum;
    }
    __syncthreads();
    if (part == 1) return;
    const float m1 = over[pair][OT * 16][lane], top = __builtin_fmaxf(m, m1), ref = top == -INF ? 0.0f : top;
    // (a wave that saw nothing has m -inf, and its factor is 0)
    const float f0 = __builtin_amdgcn_exp2f((m - ref) * a.c2), f1 = __builtin_amdgcn_exp2f((m1 - ref) * a.c2);
    sum = sum * f0 + over[pair][OT * 16 + 1][lane] * f1;
#pragma unroll
    for (int o = 0; o < OT; o++)
#pragma unroll
      for (int e = 0; e < 16; e++) out[o][e] = out[o][e] * f0 + over[pair][o * 16 + e][lane] * f1;
    m = top;
  }
  sum = sum + other_half(sum);
  if (qi >= a.sq) return;
  store_column<EL, DP>(const_cast<S *>(rows_of<EL>(a.out, b, h)) + (int64_t)qi * a.out.row, out, sum == 0.0f ? 0.0f : 1.0f / sum, a.dim);
  if (lane < 32) {
    float *lse = reinterpret_cast<float *>(const_cast<char *>(a.lse.base)) + (int64_t)b * a.lse.batch + (int64_t)h * a.lse.head + (int64_t)qi * a.lse.row;
    *lse = sum == 0.0f ? -INF : __builtin_fmaf(m, a.scale, __builtin_amdgcn_logf(sum) * LN2);
  }
}

template <class EL, int DP, int KW>
void launch_waves(nxh_context *ctx, AttentionArgs a) {
  a.tiles = (a.sq + 128 / KW - 1) / (128 / KW);
  const dim3 grid((unsigned)(a.batch * a.heads * a.tiles));
  if (a.mask.base) hipLaunchKernelGGL((attention_train_kernel<EL, DP, KW, true>), grid, dim3(256), 0, ctx->stream, a);
  else hipLaunchKernelGGL((attention_train_kernel<EL, DP, KW, false>), grid, dim3(256), 0, ctx->stream, a);
}
// Blocks of 128 queries where there are three for each unit, else of 64. Causal, us with blocks of 128 and of 64: bfloat16 [b,12,1024,64],
// b = 1, 2, 4, 5 (0.4 to 1.9 blocks of 128 a unit) 19 / 16, 20 / 17, 21 / 19, 24 / 21; 6, 7 (2.3 and 2.6) 24.4 / 25.2, 26.1 / 29.1; 8, 9, 16 (3
// to 6) 27 / 31, 29 / 36, 45 / 56; [1,32,2048,128] with 4 heads of keys (2) 70 / 56, [1,16,8192,128] (4) 303 / 341; float32 [4,8,512,64]
// (0.5) 44 / 26, [8,8,1024,64] (2) 109 / 85. The border lies between 2 and 2.3; from there to 3 the rule costs up to a tenth.
template <class EL, int DP>
void launch(nxh_context *ctx, const AttentionArgs &a) {
  const int64_t blocks = (int64_t)a.batch * a.heads * ((a.sq + 127) / 128);
  if (blocks < 3 * (ctx->compute_units > 0 ? ctx->compute_units : 256)) launch_waves<EL, DP, 2>(ctx, a);
  else launch_waves<EL, DP, 1>(ctx, a);
}
template <class EL>
void launch_dim(nxh_context *ctx, const AttentionArgs &a) {
  if (a.dim <= 32) launch<EL, 32>(ctx, a);
  else if (a.dim <= 64) launch<EL, 64>(ctx, a);
  else if (a.dim <= 96) launch<EL, 96>(ctx, a);
  else launch<EL, 128>(ctx, a);
}

}  // namespace

NXH_EXPORT int nxh_attention_train(nxh_context *ctx, const nxh_tensor *out, const nxh_tensor *lse, const nxh_tensor *q, const nxh_tensor *k,
                                   const nxh_tensor *v, const nxh_tensor *lengths, const nxh_tensor *mask, double scale, int causal) {
  NXH_DEFER_TOUCH(ctx, 2, out, lse, q, k, v, lengths, mask);
  const char *op = "attention_train";
  if (!ctx || !out || !lse || !q || !k || !v) return nxh_fail(NXH_INVALID_ARGUMENT, op, "null argument");
  int rc;
  for (const nxh_tensor *t : {out, lse, q, k, v, lengths, mask})
    if (t && (rc = nxh_check_tensor(op, t))) return rc;
  AttentionArgs a;
  if ((rc = attention_arguments(op, a, q, k, v, out, lse, lengths, mask, scale, causal, false))) return rc;
  if (a.batch == 0 || a.heads == 0 || a.sq == 0) return NXH_OK;
  for (const nxh_tensor *i : {q, k, v, lengths, mask})
    if (i && (same_start(out, i) || same_start(lse, i))) return nxh_fail(NXH_INVALID_ARGUMENT, op, "a result must not replace an input");
  if (same_start(out, lse)) return nxh_fail(NXH_INVALID_ARGUMENT, op, "two results in one place");
  std::lock_guard<std::mutex> guard(ctx->mu);
  NXH_HIP(op, hipSetDevice(ctx->device));
  nxh_set_path("attention_train");
  if (q->dtype == NXH_F32) launch_dim<gemm_tile::ElF32>(ctx, a);
  else if (q->dtype == NXH_BF16) launch_dim<gemm_tile::ElBF16>(ctx, a);
  else launch_dim<gemm_tile::ElF16>(ctx, a);
  NXH_HIP(op, hipGetLastError());
  return NXH_OK;
}
