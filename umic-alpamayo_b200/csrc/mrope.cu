// Attention input of ragged tokens in one pass: per-head RMSNorm, rotary positions with
// several axes, and the write of K and V into cache pages (umic_qk_norm_mrope_kv).
//
//   y   = x * rsqrt(mean(x^2) + eps) * w                     (per head; no weight: y = x)
//   t_i = positions[axis(i)] * inv_freq[i]                   i < rotary_dim / 2
//   out[i]     = y[i] cos t_i - y[i + r/2] sin t_i
//   out[i+r/2] = y[i+r/2] cos t_i + y[i] sin t_i             r = rotary_dim
//
// The angle is taken in 64 bits and reduced to a fraction of a turn there: in 32 bits a
// position of 30 000 leaves 2^-9 of a radian, as much as bf16's own rounding. The rest is
// fp32, rounded once on the way out. A warp owns one head row of one token.
#include <cuda_fp8.h>

#include "common.cuh"

namespace umic {
namespace {

struct MropeArgs {
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16 *q_out, *k_out;
  void *k_pages, *v_pages;
  const void *qw, *kw, *positions;
  const float *inv_freq, *k_scale, *v_scale;
  const int32_t* slots;
  uint32_t* err;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh, ko_st, ko_sh;
  int64_t p_sa, p_st, pg_sp, pg_sh, pg_ss, num_slots;
  int32_t page_size, tokens, hq, hk, d, half;
  int32_t sec[3], axes, interleaved, pos64, w_dtype, e4m3;
  float q_eps, k_eps, scaling;
};

__device__ __forceinline__ int axis_of(const MropeArgs& a, int i) {
  if (a.interleaved) {
    const int x = i % a.axes;
    return x && i < a.axes * a.sec[x] ? x : 0;
  }
  return i < a.sec[0] ? 0 : i < a.sec[0] + a.sec[1] ? 1 : 2;
}

__device__ __forceinline__ double position_of(const MropeArgs& a, int axis, int64_t t) {
  const int64_t at = axis * a.p_sa + t * a.p_st;
  return a.pos64 ? static_cast<double>(static_cast<const int64_t*>(a.positions)[at])
                 : static_cast<double>(static_cast<const int32_t*>(a.positions)[at]);
}

// cos and sin of pos * freq: the product in turns, its whole part dropped, in 64 bits
__device__ __forceinline__ void turn(double pos, float freq, float scaling, float* c, float* s) {
  const double u = pos * (static_cast<double>(freq) * 0.15915494309189533577);
  sincospif(2.f * static_cast<float>(u - rint(u)), s, c);
  *c *= scaling;
  *s *= scaling;
}

__device__ __forceinline__ void store_page(void* base, int64_t at, float x, bool e4m3, float scale) {
  if (e4m3)
    static_cast<__nv_fp8_storage_t*>(base)[at] =
        __nv_cvt_float_to_fp8(__fdiv_rn(x, scale), __NV_SATFINITE, __NV_E4M3);
  else
    static_cast<__nv_bfloat16*>(base)[at] = __float2bfloat16_rn(x);
}

__global__ void __launch_bounds__(128) mrope_kernel(MropeArgs a) {
  allow_dependent_launch();
  wait_prerequisite();
  const int lane = threadIdx.x & 31;
  const int rows = a.hq + a.hk + (a.k_pages ? a.hk : 0);
  const int64_t task = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int64_t t = task / rows;
  if (t >= a.tokens) return;
  const int r = static_cast<int>(task % rows);
  const bool is_q = r < a.hq, is_v = r >= a.hq + a.hk;
  const int h = is_q ? r : is_v ? r - a.hq - a.hk : r - a.hq;
  int64_t page_at = 0;
  if (!is_q && a.k_pages) {
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= a.num_slots) {
      if (slot != -1 && lane == 0) atomicOr(a.err, UMIC_DEVERR_BAD_PAGE);
      return;
    }
    page_at = slot / a.page_size * a.pg_sp + h * a.pg_sh + slot % a.page_size * a.pg_ss;
  }
  const __nv_bfloat16* x = is_q ? a.q + t * a.q_st + h * a.q_sh
                          : is_v ? a.v + t * a.v_st + h * a.v_sh
                                 : a.k + t * a.k_st + h * a.k_sh;
  const void* w = is_q ? a.qw : is_v ? nullptr : a.kw;
  float rstd = 1.f;
  if (w) {
    float ss = 0.f;
    for (int i = lane; i < a.d; i += 32) ss += bf(x[i]) * bf(x[i]);
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    rstd = rsqrtf(ss / static_cast<float>(a.d) + (is_q ? a.q_eps : a.k_eps));
  }
  const float* scales = is_v ? a.v_scale : a.k_scale;
  const float scale = !is_q && scales ? scales[h] : 1.f;
  auto value = [&](int i) { return w ? bf(x[i]) * rstd * load_w1(w, a.w_dtype, i) : bf(x[i]); };
  auto put = [&](int i, float y) {
    if (is_q) a.q_out[t * a.qo_st + h * a.qo_sh + i] = __float2bfloat16_rn(y);
    else if (!a.k_pages) a.k_out[t * a.ko_st + h * a.ko_sh + i] = __float2bfloat16_rn(y);
    else store_page(is_v ? a.v_pages : a.k_pages, page_at + i, y, a.e4m3, scale);
  };
  // in-place rows: a lane reads both elements of a pair before it writes either
  const int half = is_v ? 0 : a.half;
  for (int i = lane; i < half; i += 32) {
    float c, s;
    turn(position_of(a, axis_of(a, i), t), a.inv_freq[i], a.scaling, &c, &s);
    const float lo = value(i), hi = value(i + half);
    put(i, lo * c - hi * s);
    put(i + half, hi * c + lo * s);
  }
  for (int i = 2 * half + lane; i < a.d; i += 32) put(i, value(i));
}

}  // namespace
}  // namespace umic

using namespace umic;

extern "C" int umic_qk_norm_mrope_kv(
    const void* q, int64_t q_st, int64_t q_sh, int32_t hq, const void* k, int64_t k_st,
    int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh, int32_t hk, void* q_out,
    int64_t qo_st, int64_t qo_sh, void* k_out, int64_t ko_st, int64_t ko_sh,
    const void* q_weight, const void* k_weight, int w_dtype, float q_eps, float k_eps,
    const void* positions, int pos_bytes, int64_t p_sa, int64_t p_st, const float* inv_freq,
    int32_t rotary_dim, int32_t axes, int32_t s0, int32_t s1, int32_t s2, int interleaved,
    float scaling, void* k_pages, void* v_pages, int64_t pg_sp, int64_t pg_sh, int64_t pg_ss,
    int64_t num_pages, int64_t page_size, int cache_dtype, const float* k_scale,
    const float* v_scale, const int32_t* slots, int64_t tokens, int32_t head_dim,
    void* stream) {
  const char* const me = "umic_qk_norm_mrope_kv";
  clear_error();
  if (hq < 0 || hk <= 0 || tokens < 0 || head_dim <= 0)
    return fail(UMIC_ERR_INVALID_ARG, "%s: hq=%d hk=%d tokens=%lld head_dim=%d", me, hq, hk,
                (long long)tokens, head_dim);
  if (head_dim % 16 != 0 || head_dim > 256)
    return fail(UMIC_ERR_UNSUPPORTED, "%s: head_dim %d (a multiple of 16 up to 256)", me,
                head_dim);
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 16 != 0)
    return fail(UMIC_ERR_UNSUPPORTED, "%s: rotary_dim %d (a multiple of 16 up to head_dim %d)",
                me, rotary_dim, head_dim);
  if (rotary_dim > 0) {
    if (axes < 1 || axes > 3)
      return fail(UMIC_ERR_UNSUPPORTED, "%s: %d position axes (1 to 3)", me, axes);
    if (s0 < 0 || s1 < 0 || s2 < 0 || (axes < 3 && s2) || (axes < 2 && s1) ||
        static_cast<int64_t>(s0) + s1 + s2 != rotary_dim / 2)
      return fail(UMIC_ERR_INVALID_ARG, "%s: sections (%d, %d, %d) of %d axes must sum to %d", me,
                  s0, s1, s2, axes, rotary_dim / 2);
    if (pos_bytes != 4 && pos_bytes != 8)
      return fail(UMIC_ERR_INVALID_ARG, "%s: positions of %d bytes (4 or 8)", me, pos_bytes);
  }
  if (w_dtype != UMIC_DTYPE_BF16 && w_dtype != UMIC_DTYPE_FP32)
    return fail(UMIC_ERR_INVALID_ARG, "%s: bad w_dtype", me);
  if (cache_dtype != UMIC_DTYPE_BF16 && cache_dtype != UMIC_DTYPE_E4M3)
    return fail(UMIC_ERR_INVALID_ARG, "%s: bad cache_dtype", me);
  if (k_pages && (num_pages <= 0 || page_size <= 0 || page_size > 0x7fffffffLL / num_pages))
    return fail(UMIC_ERR_UNSUPPORTED, "%s: num_pages %lld x page_size %lld must stay below 2^31",
                me, (long long)num_pages, (long long)page_size);
  if (tokens > 0x7fffffffLL)
    return fail(UMIC_ERR_UNSUPPORTED, "%s: too many tokens (%lld)", me, (long long)tokens);
  if (tokens == 0) return UMIC_OK;
  if (!k || (hq > 0 && (!q || !q_out)) || (rotary_dim > 0 && (!positions || !inv_freq)) ||
      (k_pages ? !v || !v_pages || !slots : !k_out))
    return fail(UMIC_ERR_INVALID_ARG, "%s: null pointer", me);
  const int64_t pe = cache_dtype == UMIC_DTYPE_E4M3 ? 16 : 8;
  const bool q_al = hq == 0 || (aligned16(q) && aligned16(q_out) && q_st % 8 == 0 &&
                                q_sh % 8 == 0 && qo_st % 8 == 0 && qo_sh % 8 == 0);
  const bool kv_al =
      aligned16(k) && k_st % 8 == 0 && k_sh % 8 == 0 &&
      (k_pages ? aligned16(v) && v_st % 8 == 0 && v_sh % 8 == 0 && aligned16(k_pages) &&
                     aligned16(v_pages) && pg_sp % pe == 0 && pg_sh % pe == 0 && pg_ss % pe == 0
               : aligned16(k_out) && ko_st % 8 == 0 && ko_sh % 8 == 0);
  if (!q_al || !kv_al || (q_weight && !aligned16(q_weight)) || (k_weight && !aligned16(k_weight)))
    return fail(UMIC_ERR_ALIGNMENT, "%s: 16-byte alignment of bases / strides", me);
  uint32_t* err = device_error_word();
  if (!err) return fail(UMIC_ERR_DEVICE, "%s: no device error word", me);
  MropeArgs a{};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.k = static_cast<const __nv_bfloat16*>(k);
  a.v = static_cast<const __nv_bfloat16*>(v);
  a.q_out = static_cast<__nv_bfloat16*>(q_out);
  a.k_out = static_cast<__nv_bfloat16*>(k_out);
  a.k_pages = k_pages;
  a.v_pages = v_pages;
  a.qw = q_weight;
  a.kw = k_weight;
  a.positions = positions;
  a.inv_freq = inv_freq;
  a.k_scale = cache_dtype == UMIC_DTYPE_E4M3 ? k_scale : nullptr;
  a.v_scale = cache_dtype == UMIC_DTYPE_E4M3 ? v_scale : nullptr;
  a.slots = slots;
  a.err = err;
  a.q_st = q_st; a.q_sh = q_sh; a.k_st = k_st; a.k_sh = k_sh; a.v_st = v_st; a.v_sh = v_sh;
  a.qo_st = qo_st; a.qo_sh = qo_sh; a.ko_st = ko_st; a.ko_sh = ko_sh;
  a.p_sa = p_sa; a.p_st = p_st;
  a.pg_sp = pg_sp; a.pg_sh = pg_sh; a.pg_ss = pg_ss;
  a.num_slots = k_pages ? num_pages * page_size : 0;
  a.page_size = k_pages ? static_cast<int32_t>(page_size) : 1;
  a.tokens = static_cast<int32_t>(tokens);
  a.hq = hq;
  a.hk = hk;
  a.d = head_dim;
  a.half = rotary_dim / 2;
  a.sec[0] = s0; a.sec[1] = s1; a.sec[2] = s2;
  a.axes = axes;
  a.interleaved = interleaved != 0;
  a.pos64 = pos_bytes == 8;
  a.w_dtype = w_dtype;
  a.e4m3 = cache_dtype == UMIC_DTYPE_E4M3;
  a.q_eps = q_eps;
  a.k_eps = k_eps;
  a.scaling = scaling;
  const int64_t rows = static_cast<int64_t>(hq) + hk + (k_pages ? hk : 0);
  const int64_t blocks = (tokens * rows + 3) / 4;
  if (blocks > 0x7fffffffLL)
    return fail(UMIC_ERR_UNSUPPORTED, "%s: %lld tokens x %lld heads", me, (long long)tokens,
                (long long)rows);
  launch_pdl(mrope_kernel, dim3(static_cast<unsigned>(blocks)), dim3(128), 0, as_stream(stream),
             a);
  return launch_status(me);
}
