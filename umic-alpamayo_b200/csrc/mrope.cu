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
// fp32, rounded once on the way out.
//
// HBM bounds it: every row is read and written once. A group of TPH lanes owns a head row,
// 16 elements a lane: 8 of the first half and their rotary partners, so the rotation needs
// no exchange and the norm log2(TPH) shuffles. A warp takes one token and some of its row
// groups (32 / TPH rows of q, k, v in turn), the rows of two groups loaded before either is
// used. The token's angles are made once per warp, shared out among the row groups' lanes
// and handed round by shuffles: 64 sines and cosines against the 24 KB of a token's 48 rows.
#include <cuda_fp8.h>

#include <algorithm>

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
  int32_t shares, groups;  // warps of a token, row groups of each
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

// Rows read once. Not through the read-only path: q_out may be q.
__device__ __forceinline__ uint4 ld_row(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

// cos and sin of pos * freq: the product in turns, its whole part dropped, in 64 bits
__device__ __forceinline__ void turn(double pos, float freq, float scaling, float* c, float* s) {
  const double u = pos * (static_cast<double>(freq) * 0.15915494309189533577);
  sincospif(2.f * static_cast<float>(u - rint(u)), s, c);
  *c *= scaling;
  *s *= scaling;
}

// 8 values as e4m3 after a division by the scale (a true one: a product with the inverse
// would fall on the other side of a border now and then).
__device__ __forceinline__ uint2 pack8_e4m3(const float (&f)[8], float scale) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = make_float2(__fdiv_rn(f[2 * i], scale), __fdiv_rn(f[2 * i + 1], scale));
    w[i / 2] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3))
                << (i % 2 * 16);
  }
  return make_uint2(w[0], w[1]);
}

constexpr int kThreads = 256;
constexpr int kAhead = 2;  // row groups loaded before the first is used

template <int TPH, bool kE4m3>
__global__ void __launch_bounds__(kThreads) mrope_kernel(MropeArgs a) {
  allow_dependent_launch();
  wait_prerequisite();
  constexpr int kRows = 32 / TPH;     // rows of a group
  constexpr int kShare = 8 / kRows;   // angles a lane makes (TPH >= 4, so at least one)
  const int lane = threadIdx.x & 31, sub = lane % TPH, mine = lane / TPH;
  const int64_t task = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  const int t = static_cast<int>(task / a.shares);
  if (t >= a.tokens) return;
  const int rows = a.hq + a.hk + (a.k_pages ? a.hk : 0);
  const int row0 = static_cast<int>(task % a.shares) * a.groups * kRows;
  const int row1 = min(rows, row0 + a.groups * kRows);

  const int turned = a.half / 8;  // lanes of a row whose pairs are rotated
  const bool there = sub < a.d / 16, turns = sub < turned;
  const int lo = turns ? sub * 8 : 2 * a.half + (sub - turned) * 16;
  const int hi = turns ? a.half + sub * 8 : lo + 8;
  const __nv_bfloat16* const q = a.q + t * a.q_st;
  const __nv_bfloat16* const k = a.k + t * a.k_st;
  const __nv_bfloat16* const v = a.v + t * a.v_st;
  auto source = [&](int r) {
    return r < a.hq ? q + r * a.q_sh
           : r < a.hq + a.hk ? k + (r - a.hq) * a.k_sh : v + (r - a.hq - a.hk) * a.v_sh;
  };
  uint4 xl[kAhead], xh[kAhead];
  auto fetch = [&](int first) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int r = first + u * kRows + mine;
      xl[u] = xh[u] = make_uint4(0, 0, 0, 0);
      if (there && r < row1) {
        const __nv_bfloat16* p = source(r);
        xl[u] = ld_row(p + lo);
        xh[u] = ld_row(p + hi);
      }
    }
  };
  fetch(row0);

  int64_t page_at = -1;  // where the token's K and V go; -1: nowhere
  if (a.k_pages && row1 > a.hq) {
    const int slot = a.slots[t];
    if (slot >= 0 && slot < a.num_slots) {
      const int page = slot / a.page_size;
      page_at = page * a.pg_sp + (slot - page * a.page_size) * a.pg_ss;
    } else if (slot != -1 && lane == 0) {
      atomicOr(a.err, UMIC_DEVERR_BAD_PAGE);
    }
  }
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = s[i] = 0.f;
  }
  if (a.half && row0 < a.hq + a.hk) {
    float mc[kShare], ms[kShare];
#pragma unroll
    for (int x = 0; x < kShare; ++x) {
      const int i = min(sub * 8 + mine * kShare + x, a.half - 1);
      turn(position_of(a, axis_of(a, i), t), a.inv_freq[i], a.scaling, &mc[x], &ms[x]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int from = i / kShare * TPH + sub;
      const float cv = __shfl_sync(0xffffffffu, mc[i % kShare], from);
      const float sv = __shfl_sync(0xffffffffu, ms[i % kShare], from);
      c[i] = cv;
      s[i] = sv;
    }
  }

#pragma unroll 1
  for (int first = row0; first < row1; first += kAhead * kRows) {
    uint4 yl[kAhead], yh[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      yl[u] = xl[u];
      yh[u] = xh[u];
    }
    if (first + kAhead * kRows < row1) fetch(first + kAhead * kRows);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int r = first + u * kRows + mine;
      if (first + u * kRows >= row1) break;
      const bool is_q = r < a.hq, is_v = r >= a.hq + a.hk;
      const int h = is_q ? r : is_v ? r - a.hq - a.hk : r - a.hq;
      float x[8], y[8];
      unpack8(yl[u], x);
      unpack8(yh[u], y);
      if (a.qw || a.kw) {  // all lanes take part in the shuffles
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += x[i] * x[i] + y[i] * y[i];
#pragma unroll
        for (int o = TPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const void* w = is_q ? a.qw : is_v ? nullptr : a.kw;
        if (w && there) {
          const float rstd = rsqrtf(ss / static_cast<float>(a.d) + (is_q ? a.q_eps : a.k_eps));
          float wv[8];
          load_w8(w, a.w_dtype, lo, wv);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = x[i] * rstd * wv[i];
          load_w8(w, a.w_dtype, hi, wv);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = y[i] * rstd * wv[i];
        }
      }
      const bool plain = is_v || !turns;  // not "times 1 plus times 0": infinity passes
      float ox[8], oy[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ox[i] = plain ? x[i] : x[i] * c[i] - y[i] * s[i];
        oy[i] = plain ? y[i] : y[i] * c[i] + x[i] * s[i];
      }
      if (!there || r >= row1) continue;
      if (is_q || !a.k_pages) {
        __nv_bfloat16* out =
            is_q ? a.q_out + t * a.qo_st + h * a.qo_sh : a.k_out + t * a.ko_st + h * a.ko_sh;
        st_vec(out + lo, pack8(ox));
        st_vec(out + hi, pack8(oy));
      } else if (page_at >= 0) {
        const int64_t at = page_at + h * a.pg_sh;
        if constexpr (kE4m3) {
          const float* scales = is_v ? a.v_scale : a.k_scale;
          const float scale = scales ? __ldg(scales + h) : 1.f;
          uint8_t* out = static_cast<uint8_t*>(is_v ? a.v_pages : a.k_pages) + at;
          *reinterpret_cast<uint2*>(out + lo) = pack8_e4m3(ox, scale);
          *reinterpret_cast<uint2*>(out + hi) = pack8_e4m3(oy, scale);
        } else {
          __nv_bfloat16* out = static_cast<__nv_bfloat16*>(is_v ? a.v_pages : a.k_pages) + at;
          st_vec(out + lo, pack8(ox));
          st_vec(out + hi, pack8(oy));
        }
      }
    }
  }
}

template <int TPH>
void launch(const MropeArgs& a, int64_t blocks, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(blocks));
  if (a.e4m3) launch_pdl(mrope_kernel<TPH, true>, grid, dim3(kThreads), 0, st, a);
  else launch_pdl(mrope_kernel<TPH, false>, grid, dim3(kThreads), 0, st, a);
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
  const int tph = head_dim <= 64 ? 4 : head_dim <= 128 ? 8 : 16;
  const int64_t groups = (rows + 32 / tph - 1) / (32 / tph);
  // A warp each for a row group while that leaves the GPU's warps (64 an SM) unfilled; with
  // more tokens longer shares, which make a token's angles fewer times.
  const int64_t per = tokens * groups / (static_cast<int64_t>(sm_count()) * 64);
  a.groups = static_cast<int32_t>(std::max<int64_t>(1, std::min(per, groups)));
  a.shares = static_cast<int32_t>((groups + a.groups - 1) / a.groups);
  const int64_t blocks = (tokens * a.shares + kThreads / 32 - 1) / (kThreads / 32);
  if (blocks > 0x7fffffffLL)
    return fail(UMIC_ERR_UNSUPPORTED, "%s: %lld tokens x %lld heads", me, (long long)tokens,
                (long long)rows);
  cudaStream_t st = as_stream(stream);
  if (tph == 4) launch<4>(a, blocks, st);
  else if (tph == 8) launch<8>(a, blocks, st);
  else launch<16>(a, blocks, st);
  return launch_status(me);
}
