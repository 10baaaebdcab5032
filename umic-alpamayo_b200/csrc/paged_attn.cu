// Attention of one new token per request over its key-value pages (umic_paged_attention).
//
//   out[b, h] = sum_j softmax_j(scale q[b, h] . k_j) v_j,  j < kv_lens[b]
//
// One pass over K and V with a running maximum m and sum l: at a new score s,
// m' = max(m, s), and the sum and the output accumulator are multiplied by
// exp(m - m') before exp(s - m') and exp(s - m') v are added. A warp owns one query head.
#include <cuda_fp8.h>

#include <cmath>

#include "common.cuh"

namespace umic {
namespace {

struct PagedArgs {
  const __nv_bfloat16* q;
  const void *k_pages, *v_pages;
  const float *k_scale, *v_scale;
  const int32_t *table, *lens;
  __nv_bfloat16* out;
  float* lse;
  uint32_t* err;
  int64_t q_sb, q_sh, pg_sp, pg_sh, pg_ss, table_stride, max_len, num_pages, o_sb, o_sh;
  int32_t page_size, hq, hkv, batch;
  float scale;
};

__device__ __forceinline__ float load_elem(const void* p, int64_t at, bool e4m3) {
  if (!e4m3) return bf(static_cast<const __nv_bfloat16*>(p)[at]);
  const __half_raw h =
      __nv_cvt_fp8_to_halfraw(static_cast<const __nv_fp8_storage_t*>(p)[at], __NV_E4M3);
  return __half2float(__half(h));
}

template <int D, bool kE4m3>
__global__ void __launch_bounds__(32) paged_attn_kernel(PagedArgs a) {
  allow_dependent_launch();
  wait_prerequisite();
  constexpr int kPer = (D + 31) / 32;
  const int lane = threadIdx.x;
  const int b = blockIdx.x / a.hq, h = blockIdx.x % a.hq, hk = h / (a.hq / a.hkv);
  int64_t len = a.lens[b];
  if (len > a.max_len || len < 0) {
    if (lane == 0) atomicOr(a.err, UMIC_DEVERR_BAD_PAGE);
    len = len < 0 ? 0 : a.max_len;
  }
  float q[kPer], o[kPer];
  for (int i = 0; i < kPer; ++i) {
    const int e = lane + 32 * i;
    q[i] = e < D ? bf(a.q[b * a.q_sb + h * a.q_sh + e]) : 0.f;
    o[i] = 0.f;
  }
  const float scale = a.scale * (a.k_scale ? a.k_scale[hk] : 1.f);
  float m = -INFINITY, l = 0.f;
  for (int64_t j = 0; j < len; ++j) {
    const int64_t page = a.table[b * a.table_stride + j / a.page_size];
    if (page < 0 || page >= a.num_pages) {
      if (lane == 0) atomicOr(a.err, UMIC_DEVERR_BAD_PAGE);
      continue;
    }
    const int64_t at = page * a.pg_sp + hk * a.pg_sh + j % a.page_size * a.pg_ss;
    float s = 0.f;
    for (int i = 0; i < kPer; ++i) {
      const int e = lane + 32 * i;
      if (e < D) s += q[i] * load_elem(a.k_pages, at + e, kE4m3);
    }
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= scale;
    const float top = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.f : expf(m - top);
    const float p = top == -INFINITY ? 0.f : expf(s - top);
    m = top;
    l = l * keep + p;
    for (int i = 0; i < kPer; ++i) {
      const int e = lane + 32 * i;
      if (e < D) o[i] = o[i] * keep + p * load_elem(a.v_pages, at + e, kE4m3);
    }
  }
  const float inv = l == 0.f ? 0.f : (a.v_scale ? a.v_scale[hk] : 1.f) / l;
  for (int i = 0; i < kPer; ++i) {
    const int e = lane + 32 * i;
    if (e < D) a.out[b * a.o_sb + h * a.o_sh + e] = __float2bfloat16_rn(o[i] * inv);
  }
  if (a.lse && lane == 0)
    a.lse[static_cast<int64_t>(b) * a.hq + h] = l == 0.f ? -INFINITY : m + logf(l);
}

template <int D>
void launch_d(const PagedArgs& a, bool e4m3, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(a.batch) * a.hq);
  if (e4m3) launch_pdl(paged_attn_kernel<D, true>, grid, dim3(32), 0, st, a);
  else launch_pdl(paged_attn_kernel<D, false>, grid, dim3(32), 0, st, a);
}

}  // namespace
}  // namespace umic

using namespace umic;

extern "C" size_t umic_paged_attention_workspace_bytes(int32_t, int32_t, int32_t) { return 16; }

extern "C" int umic_paged_attention(
    const void* q, int64_t q_sb, int64_t q_sh, const void* k_pages, const void* v_pages,
    int64_t pg_sp, int64_t pg_sh, int64_t pg_ss, int64_t num_pages, int64_t page_size,
    int cache_dtype, const float* k_scale, const float* v_scale, const int32_t* block_table,
    int64_t table_stride, int64_t max_pages, const int32_t* kv_lens, void* out, int64_t o_sb,
    int64_t o_sh, float* lse, int64_t batch, int32_t hq, int32_t hkv, int32_t head_dim,
    float scale, void* workspace, size_t workspace_bytes, void* stream) {
  const char* const me = "umic_paged_attention";
  clear_error();
  if (batch < 0 || hq <= 0 || hkv <= 0 || num_pages <= 0 || page_size <= 0 || max_pages < 0)
    return fail(UMIC_ERR_INVALID_ARG,
                "%s: batch=%lld hq=%d hkv=%d num_pages=%lld page_size=%lld max_pages=%lld", me,
                (long long)batch, hq, hkv, (long long)num_pages, (long long)page_size,
                (long long)max_pages);
  if (cache_dtype != UMIC_DTYPE_BF16 && cache_dtype != UMIC_DTYPE_E4M3)
    return fail(UMIC_ERR_INVALID_ARG, "%s: bad cache_dtype", me);
  if (hq % hkv != 0)
    return fail(UMIC_ERR_UNSUPPORTED, "%s: %d query heads over %d KV heads", me, hq, hkv);
  if (head_dim != 64 && head_dim != 80 && head_dim != 96 && head_dim != 128 && head_dim != 256)
    return fail(UMIC_ERR_UNSUPPORTED, "%s: head_dim %d (64, 80, 96, 128 or 256)", me, head_dim);
  if (page_size % 16 != 0)
    return fail(UMIC_ERR_UNSUPPORTED, "%s: page_size %lld (a multiple of 16)", me,
                (long long)page_size);
  if (page_size > 0x7fffffffLL / num_pages ||
      (max_pages > 0 && page_size > 0x7fffffffLL / max_pages) || batch > 0x7fffffffLL / hq)
    return fail(UMIC_ERR_UNSUPPORTED,
                "%s: num_pages * page_size, max_pages * page_size and batch * hq must stay below "
                "2^31",
                me);
  if (batch == 0) return UMIC_OK;
  if (!q || !k_pages || !v_pages || !kv_lens || !out || (max_pages > 0 && !block_table))
    return fail(UMIC_ERR_INVALID_ARG, "%s: null pointer", me);
  const int64_t pe = cache_dtype == UMIC_DTYPE_E4M3 ? 16 : 8;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out) ||
      q_sb % 8 || q_sh % 8 || o_sb % 8 || o_sh % 8 || pg_sp % pe || pg_sh % pe || pg_ss % pe)
    return fail(UMIC_ERR_ALIGNMENT, "%s: 16-byte alignment of bases / strides", me);
  if (!workspace || !aligned16(workspace) ||
      workspace_bytes < umic_paged_attention_workspace_bytes(hq, hkv, head_dim))
    return fail(UMIC_ERR_INVALID_ARG, "%s: workspace of %zu bytes (%zu needed, 16-byte aligned)",
                me, workspace_bytes, umic_paged_attention_workspace_bytes(hq, hkv, head_dim));
  uint32_t* err = device_error_word();
  if (!err) return fail(UMIC_ERR_DEVICE, "%s: no device error word", me);
  const bool e4m3 = cache_dtype == UMIC_DTYPE_E4M3;
  PagedArgs a{static_cast<const __nv_bfloat16*>(q), k_pages, v_pages, e4m3 ? k_scale : nullptr,
              e4m3 ? v_scale : nullptr, block_table, kv_lens,
              static_cast<__nv_bfloat16*>(out), lse, err, q_sb, q_sh, pg_sp, pg_sh, pg_ss,
              table_stride, max_pages * page_size, num_pages, o_sb, o_sh,
              static_cast<int32_t>(page_size), hq, hkv, static_cast<int32_t>(batch), scale};
  cudaStream_t st = as_stream(stream);
  if (head_dim == 64) launch_d<64>(a, e4m3, st);
  else if (head_dim == 80) launch_d<80>(a, e4m3, st);
  else if (head_dim == 96) launch_d<96>(a, e4m3, st);
  else if (head_dim == 128) launch_d<128>(a, e4m3, st);
  else launch_d<256>(a, e4m3, st);
  return launch_status(me);
}
