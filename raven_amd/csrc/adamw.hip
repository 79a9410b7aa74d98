// adamw.hip — nxh_adamw: one step of AdamW over all tensors of a model. For each element, with t the step's number,
//   m = b1 m + (1 - b1) f g,  v = b2 v + (1 - b2) (f g)^2
//   w = w (1 - lr decay) - lr / (1 - b1^t) m / (sqrt v / sqrt(1 - b2^t) + eps)
// lr, t and f come from device memory, so that a recorded step goes on counting. Every product and sum is a float32 rounding of
// its own; what belongs to a step (1 - b^t) is made in float64. A 16-bit parameter is w rounded once.
//
// States of 8 bits: m and sqrt v as e4m3 codes of up to 448, each block of 256 elements with a float32 scale of its own. The
// codes lie 6 to 12 % apart, and a step moves v by some 0.1 %: rounded to nearest it would stand still. So each is rounded
// to one of its two neighbours by 16 random bits (Threefry of the key and the element's place among all blocks of the
// call; sqrt v's are m's with their bytes swapped), whose mean is the value. sqrt v is never rounded to zero: m / eps would
// be what follows. A step's own update uses m and v as they are before they are rounded.
//
// What bounds it: memory, 28 bytes an element in float32. GPT-2's tensors, 196 with projections apart (124 million elements, bfloat16 with masters) take 675 us
// in four launches, 5.2 TB/s, with states of 8 bits 444 to 448 us in five, 4.5 TB/s; a few small ones 13 us, of which the device has 7.
// A launch takes as many tensors as its arguments hold; a block finds its tensor among them by halving. A lane requests all that it
// will change before it makes the step's factors.

#include "lane_groups.hpp"
#include "threefry.hpp"

namespace {

constexpr int EACH = 8, TURNS = 2, CHUNK = 256 * EACH * TURNS;  // elements of a lane at once, and of a block
constexpr int SCALE = 256;                                      // elements of a scale

template <int BITS>
struct AdamwTensor {
  char *p;
  const char *g;
  char *m, *v;
  float *w;
  int64_t n;
};
template <>
struct AdamwTensor<8> {
  char *p;
  const char *g;
  char *m, *v;
  float *w;
  int64_t n;
  float *m_scales, *v_scales;
  int64_t before;  // scales of the call's tensors before this one
};
template <int BITS>
struct AdamwArgs {
  static constexpr int MANY = BITS == 8 ? 48 : 64;
  AdamwTensor<BITS> t[MANY];
  uint32_t first[MANY + 1];  // block of the launch
  int count;
  const float *rate, *factor;
  const int32_t *step, *key;
  int64_t key_step;
  double beta1, beta2, decay;
  float eps;
};
static_assert(sizeof(AdamwArgs<8>) <= 3840 && sizeof(AdamwArgs<32>) <= 3840, "kernel arguments of 4 KB");

// x^n, n >= 0.
__device__ __forceinline__ double power(double x, int n) {
  double y = 1.0;
  for (; n; n >>= 1, x = x * x)
    if (n & 1) y = y * x;
  return y;
}

// EACH elements from i on; `left` of them exist, the others are zeros.
template <int DT>
__device__ __forceinline__ void load_each(const char *base, int64_t i, int left, float (&x)[EACH]) {
  using IO = Io<DT>;
  using S = typename IO::S;
  const S *p = reinterpret_cast<const S *>(base) + i;
  if (left >= EACH) {
#pragma unroll
    for (int k = 0; k < EACH / IO::V; k++) {
      float y[IO::V];
      IO::widen(load_words(p + k * IO::V), y);
#pragma unroll
      for (int j = 0; j < IO::V; j++) x[k * IO::V + j] = y[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < EACH; j++) x[j] = j < left ? IO::ld(p[j]) : 0.0f;
  }
}
template <int DT>
__device__ __forceinline__ void store_each(char *base, int64_t i, int left, const float (&x)[EACH]) {
  using IO = Io<DT>;
  using S = typename IO::S;
  S *p = reinterpret_cast<S *>(base) + i;
  if (left >= EACH) {
#pragma unroll
    for (int k = 0; k < EACH / IO::V; k++) {
      float y[IO::V];
#pragma unroll
      for (int j = 0; j < IO::V; j++) y[j] = x[k * IO::V + j];
      store_words(p + k * IO::V, IO::narrow(y));
    }
  } else {
#pragma unroll
    for (int j = 0; j < EACH; j++)
      if (j < left) p[j] = IO::st(x[j]);
  }
}

// Codes of EACH elements, and back.
__device__ __forceinline__ uint2 load_codes(const char *base, int64_t i, int left) {
  uint2 c = {0, 0};
  if (left >= EACH) {
    __builtin_memcpy(&c, base + i, EACH);
  } else {
#pragma unroll
    for (int j = 0; j < EACH; j++)
      if (j < left) (j < 4 ? c.x : c.y) |= (uint32_t)(uint8_t)base[i + j] << (8 * (j & 3));
  }
  return c;
}
__device__ __forceinline__ void store_codes(char *base, int64_t i, int left, uint2 c) {
  if (left >= EACH) {
    __builtin_memcpy(base + i, &c, EACH);
  } else {
#pragma unroll
    for (int j = 0; j < EACH; j++)
      if (j < left) base[i + j] = (char)((j < 4 ? c.x : c.y) >> (8 * (j & 3)));
  }
}
__device__ __forceinline__ void decode(uint2 c, float scale, float (&x)[EACH]) {
#pragma unroll
  for (int h = 0; h < 4; h++) {
    const uint32_t w = h < 2 ? c.x : c.y;
    const auto two = h & 1 ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    x[2 * h] = two[0] * scale;
    x[2 * h + 1] = two[1] * scale;
  }
}
// The code of x, y = |x| of the block's largest times 448: one of its two neighbours, the upper with probability of its distance from
// the lower. Below 2^-6 codes are 2^-9 apart, as they are from 2^-6 on, where they are rounded.
template <bool NEVER_ZERO>
__device__ __forceinline__ uint32_t code_of(float x, float y, uint32_t u) {
  const bool low = y < 0x1p-6f;
  const uint32_t bits = f2u(low ? y + 0x1p-6f : y) + (u << 4);
  uint32_t c = (bits >> 20) - (low ? 968u : 960u);
  c = c < 0x7eu ? c : 0x7eu;
  if (NEVER_ZERO) c = y > 0.0f && c == 0 ? 1u : c;
  c = y != y ? 0x7fu : c;
  return c | (f2u(x) >> 31) << 7;
}
// Codes of the EACH elements of each of 32 lanes, which are a block, and its scale.
template <bool NEVER_ZERO>
__device__ __forceinline__ uint2 encode(const float (&x)[EACH], const uint32_t (&u)[EACH], float &scale) {
  float most = 0.0f;
#pragma unroll
  for (int j = 0; j < EACH; j++) most = __builtin_fmaxf(most, __builtin_fabsf(x[j]));
  most = lanes_combine<32>(most, [](float a, float b) { return __builtin_fmaxf(a, b); });
  const bool some = most >= 0x1p-100f;
  const float inverse = some ? (1.0f / most) * 448.0f : 0.0f;
  scale = some ? most * (float)(1.0 / 448.0) : 0.0f;
  uint2 c = {0, 0};
#pragma unroll
  for (int j = 0; j < EACH; j++) (j < 4 ? c.x : c.y) |= code_of<NEVER_ZERO>(x[j], __builtin_fabsf(x[j]) * inverse, u[j]) << (8 * (j & 3));
  return c;
}

template <int DT, bool MASTERS, int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(AdamwArgs<BITS> a) {
  int low = 0, high = a.count;  // the tensor whose blocks this one is among
  while (high - low > 1) {
    const int mid = (low + high) / 2;
    if (blockIdx.x >= a.first[mid]) low = mid;
    else high = mid;
  }
  const AdamwTensor<BITS> t = a.t[low];
  const int64_t begin = (int64_t)(blockIdx.x - a.first[low]) * CHUNK;

  float g[TURNS][EACH], w[TURNS][EACH], m[TURNS][EACH], v[TURNS][EACH];
  int left[TURNS];
#pragma unroll
  for (int k = 0; k < TURNS; k++) {
    const int64_t i = begin + (k * 256 + threadIdx.x) * EACH;
    left[k] = (int)(t.n - i < EACH ? t.n - i : EACH);
    load_each<DT>(t.g, i, left[k], g[k]);
    if constexpr (MASTERS) load_each<NXH_F32>(reinterpret_cast<const char *>(t.w), i, left[k], w[k]);
    else load_each<DT>(t.p, i, left[k], w[k]);
    if constexpr (BITS == 32) {
      load_each<NXH_F32>(t.m, i, left[k], m[k]);
      load_each<NXH_F32>(t.v, i, left[k], v[k]);
    } else {
      const uint2 mc = load_codes(t.m, i, left[k]), vc = load_codes(t.v, i, left[k]);
      decode(mc, left[k] > 0 ? t.m_scales[i / SCALE] : 0.0f, m[k]);
      decode(vc, left[k] > 0 ? t.v_scales[i / SCALE] : 0.0f, v[k]);
#pragma unroll
      for (int j = 0; j < EACH; j++) v[k][j] = v[k][j] * v[k][j];
    }
  }
  const int step = a.step[0] > 1 ? a.step[0] : 1;
  const double rate = (double)a.rate[0];
  const float shrink = (float)(1.0 - rate * a.decay), size = (float)(rate / (1.0 - power(a.beta1, step)));
  const float root = (float)(1.0 / __builtin_sqrt(1.0 - power(a.beta2, step)));
  const float factor = a.factor ? a.factor[0] : 1.0f;
  const float b1 = (float)a.beta1, c1 = (float)(1.0 - a.beta1), b2 = (float)a.beta2, c2 = (float)(1.0 - a.beta2);
#pragma unroll
  for (int k = 0; k < TURNS; k++) {
    const int64_t i = begin + (k * 256 + threadIdx.x) * EACH;
    float r[EACH];
#pragma unroll
    for (int j = 0; j < EACH; j++) {
      const float x = g[k][j] * factor;
      m[k][j] = m[k][j] * b1 + x * c1;
      v[k][j] = v[k][j] * b2 + x * x * c2;
      r[j] = __builtin_sqrtf(v[k][j]);
      w[k][j] = w[k][j] * shrink - m[k][j] / (r[j] * root + a.eps) * size;
    }
    if constexpr (MASTERS) store_each<NXH_F32>(reinterpret_cast<char *>(t.w), i, left[k], w[k]);
    store_each<DT>(t.p, i, left[k], w[k]);
    if constexpr (BITS == 32) {
      store_each<NXH_F32>(t.m, i, left[k], m[k]);
      store_each<NXH_F32>(t.v, i, left[k], v[k]);
    } else {
      uint32_t u[EACH], z[EACH];
#pragma unroll
      for (int q = 0; q < EACH / 4; q++) {
        const uint64_t block = (uint64_t)(t.before * SCALE + i) / 4 + q;
        uint32_t w0 = (uint32_t)block, w1 = (uint32_t)(block >> 32);
        threefry_block((uint32_t)a.key[0], (uint32_t)a.key[a.key_step], w0, w1);
        u[4 * q] = w0 & 0xffffu, u[4 * q + 1] = w0 >> 16, u[4 * q + 2] = w1 & 0xffffu, u[4 * q + 3] = w1 >> 16;
      }
#pragma unroll
      for (int j = 0; j < EACH; j++) z[j] = (u[j] << 8 | u[j] >> 8) & 0xffffu;
      float m_scale, v_scale;
      const uint2 mc = encode<false>(m[k], u, m_scale), vc = encode<true>(r, z, v_scale);
      store_codes(t.m, i, left[k], mc);
      store_codes(t.v, i, left[k], vc);
      if ((threadIdx.x & 31) == 0 && left[k] > 0) {
        t.m_scales[i / SCALE] = m_scale;
        t.v_scales[i / SCALE] = v_scale;
      }
    }
  }
}

// ── host side ───────────────────────────────────────────────────────────────
int64_t elements(const nxh_tensor *t) {
  int64_t n = 1;
  for (int d = 0; d < t->ndim; d++) n *= t->shape[d];
  return n;
}
bool dense(const nxh_tensor *t) {
  if (elements(t) == 0) return true;
  int64_t step = 1;
  for (int d = t->ndim - 1; d >= 0; d--) {
    if (t->shape[d] > 1 && t->strides[d] != step) return false;
    step *= t->shape[d];
  }
  return true;
}
char *start_of(const nxh_tensor *t) { return (char *)t->data + t->offset * (int64_t)nxh_elem_size(t->dtype); }

struct AdamwCall {
  int count, dt;
  const nxh_tensor *const *p, *const *g, *const *m, *const *v, *const *w, *const *m_scales, *const *v_scales;
};

template <int DT, bool MASTERS, int BITS>
void launch(nxh_context *ctx, const AdamwCall &c, AdamwArgs<BITS> &a) {
  int64_t before = 0;
  for (int i = 0; i < c.count;) {
    a.count = 0;
    a.first[0] = 0;
    int64_t blocks = 0;
    for (; i < c.count && a.count < AdamwArgs<BITS>::MANY; i++) {
      const int64_t n = elements(c.p[i]), own = (n + CHUNK - 1) / CHUNK;
      if (n == 0) continue;
      if (blocks > 0 && blocks + own > 0x7fffffff) break;
      AdamwTensor<BITS> &t = a.t[a.count];
      t.p = start_of(c.p[i]);
      t.g = start_of(c.g[i]);
      t.m = start_of(c.m[i]);
      t.v = start_of(c.v[i]);
      t.w = MASTERS ? (float *)start_of(c.w[i]) : nullptr;
      t.n = n;
      if constexpr (BITS == 8) {
        t.m_scales = (float *)start_of(c.m_scales[i]);
        t.v_scales = (float *)start_of(c.v_scales[i]);
        t.before = before;
        before += (n + SCALE - 1) / SCALE;
      }
      blocks += own;
      a.first[++a.count] = (uint32_t)blocks;
    }
    if (blocks > 0) hipLaunchKernelGGL((adamw_kernel<DT, MASTERS, BITS>), dim3((unsigned)blocks), dim3(256), 0, ctx->stream, a);
  }
}
template <int BITS>
void launch_dtype(nxh_context *ctx, const AdamwCall &c, AdamwArgs<BITS> &a) {
  if (c.dt == NXH_F32) launch<NXH_F32, false, BITS>(ctx, c, a);
  else if (c.dt == NXH_BF16 && c.w) launch<NXH_BF16, true, BITS>(ctx, c, a);
  else if (c.dt == NXH_BF16) launch<NXH_BF16, false, BITS>(ctx, c, a);
  else if (c.w) launch<NXH_F16, true, BITS>(ctx, c, a);
  else launch<NXH_F16, false, BITS>(ctx, c, a);
}
bool one_of(const nxh_tensor *t, int dtype) { return t->dtype == dtype && elements(t) == 1; }

}  // namespace

NXH_EXPORT int nxh_adamw(nxh_context *ctx, int count, const nxh_tensor *const *params, const nxh_tensor *const *grads,
                         const nxh_tensor *const *m, const nxh_tensor *const *v, const nxh_tensor *const *masters,
                         const nxh_tensor *const *m_scales, const nxh_tensor *const *v_scales, const nxh_tensor *rate,
                         const nxh_tensor *step, const nxh_tensor *factor, const nxh_tensor *key, double beta1, double beta2,
                         double eps, double decay) {
  NXH_DEFER_BARRIER(ctx);
  const char *op = "adamw";
  if (!ctx || count < 0 || !rate || !step || (count > 0 && (!params || !grads || !m || !v)) || (!m_scales) != (!v_scales) || (!m_scales) != (!key))
    return nxh_fail(NXH_INVALID_ARGUMENT, op, "null argument");
  int rc;
  const int bits = m_scales ? 8 : 32;
  const int dt = count > 0 && params[0] ? params[0]->dtype : NXH_F32;
  if (dt != NXH_F32 && dt != NXH_BF16 && dt != NXH_F16) return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
  if (masters && dt == NXH_F32) return nxh_fail(NXH_INVALID_ARGUMENT, op, "float32 parameters need no masters");
  for (const nxh_tensor *t : {rate, step, factor, key})
    if (t && (rc = nxh_check_tensor(op, t))) return rc;
  if (!one_of(rate, NXH_F32) || (factor && !one_of(factor, NXH_F32))) return nxh_fail(NXH_INVALID_ARGUMENT, op, "rate and factor must be one float32");
  if (!one_of(step, NXH_I32)) return nxh_fail(NXH_INVALID_ARGUMENT, op, "step must be one int32");
  if (key && (key->dtype != NXH_I32 || key->ndim != 1 || key->shape[0] != 2)) return nxh_fail(NXH_INVALID_ARGUMENT, op, "key must be two int32");
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0)) return nxh_fail(NXH_INVALID_ARGUMENT, op, "beta1 and beta2 must be at least 0 and below 1");
  if (!(eps >= 0.0) || !(decay >= 0.0)) return nxh_fail(NXH_INVALID_ARGUMENT, op, "eps and decay must be >= 0");
  struct Range {
    const char *begin, *end;
    bool written;
  };
  std::vector<Range> ranges;  // (all its room is taken here)
  try {
    ranges.reserve((size_t)count * (4 + (masters ? 1 : 0) + (m_scales ? 2 : 0)) + 4);
  } catch (const std::bad_alloc &) {
    return nxh_fail(NXH_FAILURE, op, "out of host memory");
  }
  for (int i = 0; i < count; i++) {
    const nxh_tensor *all[] = {params[i], grads[i], m[i], v[i], masters ? masters[i] : nullptr, m_scales ? m_scales[i] : nullptr, v_scales ? v_scales[i] : nullptr};
    const int kinds[] = {dt, dt, bits == 8 ? NXH_F8E4M3 : NXH_F32, bits == 8 ? NXH_F8E4M3 : NXH_F32, NXH_F32, NXH_F32, NXH_F32};
    for (int k = 0; k < 7; k++) {
      const bool wanted = k < 4 || (k == 4 ? masters != nullptr : m_scales != nullptr);
      if (!wanted) continue;
      const nxh_tensor *t = all[k];
      if (!t) return nxh_fail(NXH_INVALID_ARGUMENT, op, "null argument");
      if ((rc = nxh_check_tensor(op, t))) return rc;
      if (t->dtype != kinds[k]) return nxh_fail(NXH_FAILURE, op, NXH_ERR_UNSUPPORTED);
      if (k < 5 ? !nxh_same_shape(t, params[i]) : t->ndim != 1 || t->shape[0] != (elements(params[i]) + SCALE - 1) / SCALE)
        return nxh_fail(NXH_INVALID_ARGUMENT, op, NXH_ERR_SHAPE);
      if (!dense(t)) return nxh_fail(NXH_FAILURE, op, "tensors must be contiguous");
      if (elements(t) > 0) ranges.push_back({start_of(t), start_of(t) + elements(t) * (int64_t)nxh_elem_size(t->dtype), k != 1});
    }
  }
  for (const nxh_tensor *t : {rate, step, factor, key}) {  // of one or two elements of 4 bytes
    if (!t) continue;
    const char *at = start_of(t);
    const int64_t to = t == key ? t->strides[0] * 4 : 0;
    ranges.push_back({at + std::min<int64_t>(0, to), at + std::max<int64_t>(0, to) + 4, false});
  }
  std::sort(ranges.begin(), ranges.end(), [](const Range &x, const Range &y) { return x.begin < y.begin; });
  const char *end = nullptr, *written_end = nullptr;  // of the ranges so far, and of those that are written
  for (const Range &r : ranges) {
    if (r.begin < (r.written ? end : written_end)) return nxh_fail(NXH_INVALID_ARGUMENT, op, "a tensor that is written appears twice");
    end = std::max(end, r.end);
    if (r.written) written_end = std::max(written_end, r.end);
  }
  if (nxh_defer_active(ctx))  // a deferred window may take a tensor's old contents for a constant
    for (const nxh_tensor *const *written : {params, m, v, masters, m_scales, v_scales})
      if (written) nxh_defer_written(ctx, written, count);
  const AdamwCall c = {count, dt, params, grads, m, v, masters, m_scales, v_scales};
  auto fill = [&](auto &a) {
    a.rate = (const float *)start_of(rate);
    a.factor = factor ? (const float *)start_of(factor) : nullptr;
    a.step = (const int32_t *)start_of(step);
    a.key = key ? (const int32_t *)start_of(key) : nullptr;
    a.key_step = key ? key->strides[0] : 0;
    a.beta1 = beta1;
    a.beta2 = beta2;
    a.decay = decay;
    a.eps = (float)eps;
  };
  std::lock_guard<std::mutex> guard(ctx->mu);
  NXH_HIP(op, hipSetDevice(ctx->device));
  nxh_set_path(bits == 8 ? "adamw_8bit" : "adamw");
  if (bits == 8) {
    AdamwArgs<8> a;
    fill(a);
    launch_dtype<8>(ctx, c, a);
  } else {
    AdamwArgs<32> a;
    fill(a);
    launch_dtype<32>(ctx, c, a);
  }
  NXH_HIP(op, hipGetLastError());
  return NXH_OK;
}
