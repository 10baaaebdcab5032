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
// HBM bounds it: every row is read and written once, 24 KB for a token of 32 + 8 + 8 heads,
// and the issue slots run close behind, so the work per row is kept small. A group of TPH
// lanes owns a head row, 16 elements a lane: 8 of the first half and their rotary partners,
// so the rotation needs no exchange and the norm log2(TPH) shuffles. The row groups (32 / TPH
// rows of one kind: q, k or v) of all tokens form one line, and every resident warp walks
// over an equal run of it; each lane copies its own pieces of the next kDepth groups, across
// tokens, into shared memory with asynchronous loads. A token's angles are made once per warp,
// shared out among the row groups' lanes and handed round by shuffles, times the norm's
// weights, when the warp comes to the q rows and to the k rows:
//   out[i] = rstd (x[i] w[i] cos - x[i + r/2] w[i + r/2] sin), and so on.
// Measured: 24800 tokens of 32 + 8 + 8 heads x 128 into e4m3 pages 103 us (0.83 of measured
// HBM), 3100 into bf16 pages 14.5 us (0.80), 6200 tokens appended as they are 9.7 us (0.80),
// into e4m3 pages 11.5 us (0.50), 24800 of them 33 us (0.71), 8 tokens 3.2 us. 16384 x (16 +
// 16) x 80 without norm or cache 37.5 us (0.68): latency, at the 16 warps an SM that 128
// registers allow (issue slots 0.62 busy, DRAM 0.40; the angles' products are made for q and
// again for k, and a sixth of the lanes holds no row). (Whole tokens or shares of one to a warp
// instead of equal runs: 108 and 17.7 us for the first two, while the first took 101.)
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
  int64_t run;      // row groups of a warp,
  int32_t longer;   // one more for the first so many
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

__device__ __forceinline__ double position_at(const MropeArgs& a, int64_t at) {
  return a.pos64 ? static_cast<double>(static_cast<const int64_t*>(a.positions)[at])
                 : static_cast<double>(static_cast<const int32_t*>(a.positions)[at]);
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

// cos and sin of pos * turns a position: the product in turns, its whole part dropped, in
// 64 bits
__device__ __forceinline__ void turn(double pos, double turns, float scaling, float* c, float* s) {
  const double u = pos * turns;
  sincospif(2.f * static_cast<float>(u - rint(u)), s, c);
  *c *= scaling;
  *s *= scaling;
}

__device__ __forceinline__ uint2 pack8_e4m3(const float (&f)[8]) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i / 2] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(
                    make_float2(f[2 * i], f[2 * i + 1]), __NV_SATFINITE, __NV_E4M3))
                << (i % 2 * 16);
  return make_uint2(w[0], w[1]);
}

// A lane's values over the scale of their head, for e4m3. The product with the scale's
// rounded inverse alone carries some quotients over the border between two e4m3 values; its
// remainder, times the inverse again (Markstein's correction, 1990), puts it right for less
// than a division: 24800 tokens of 32 + 8 + 8 heads take 101 us with the product, 103 us so
// and 118 us with divisions, 24800 appended as they are 27, 33 and 45 us. Before its last
// rounding the quotient is off by 2^-46 of itself; the quotients of bf16 values (above
// 2^-100, where the remainder is normal) come no nearer to the middle between a border and
// the float beside it, so they are stored as after a division, bit for bit.
__device__ __forceinline__ void divide(float (&x)[8], float (&y)[8], float scale) {
  const float inv = 1.f / scale;
  auto over = [scale, inv](float v) {
    // 512 saturates all the same, and the remainder of an infinity would be NaN
    const float q = fminf(fmaxf(v * inv, -512.f), 512.f);
    return fmaf(-fmaf(q, scale, -v), inv, q);  // so signed, -0 stays -0
  };
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = over(x[i]);
    y[i] = over(y[i]);
  }
}

// The sum over a row's lanes.
template <int TPH>
__device__ __forceinline__ float row_sum(float x, int mine) {
  if constexpr ((TPH & (TPH - 1)) == 0) {
#pragma unroll
    for (int o = TPH / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
  }
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < TPH; ++j) sum += __shfl_sync(0xffffffffu, x, min(mine * TPH + j, 31));
  return sum;
}

constexpr int kThreads = 256;
// CTAs per SM: what their registers allow (a write without norm and rotation needs half).
constexpr int blocks_per_sm(bool work) { return work ? 2 : 4; }
constexpr int kDepth = 4;  // row groups of a warp under way, 1 KB each

// TPH lanes hold a row; kWork: something is normed or rotated.
template <int TPH, bool kE4m3, bool kWork>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(kWork)) mrope_kernel(MropeArgs a) {
  __shared__ uint4 s_rows[kThreads / 32][kDepth][2][32];  // read by the lane that copied
  allow_dependent_launch();
  wait_prerequisite();
  constexpr int kRows = 32 / TPH;                   // rows of a group
  constexpr int kShare = (8 + kRows - 1) / kRows;   // angles a lane makes
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % TPH, mine = lane / TPH;
  const int64_t worker = blockIdx.x * (kThreads / 32) + warp;
  const int k_from = (a.hq + kRows - 1) / kRows, v_from = k_from + (a.hk + kRows - 1) / kRows;
  const int all = a.k_pages ? 2 * v_from - k_from : v_from;  // row groups, q before k before v
  const int64_t begin_at = worker * a.run + min(worker, static_cast<int64_t>(a.longer));
  int run = static_cast<int>(a.run + (worker < a.longer));  // still to do
  if (run <= 0) return;
  const int first = static_cast<int>(
      begin_at >> 32 ? begin_at / all : static_cast<uint32_t>(begin_at) / static_cast<uint32_t>(all));
  const int first_group = static_cast<int>(begin_at - static_cast<int64_t>(first) * all);

  const int turned = a.half / 8;  // lanes of a row whose pairs are rotated
  const bool there = mine < kRows && sub < a.d / 16, turns = kWork && sub < turned;
  // the rest of the row in two runs as well, so that lanes side by side copy side by side
  const int lo = sub < turned ? sub * 8 : 2 * a.half + (sub - turned) * 8;
  const int hi = lo + (sub < turned ? a.half : a.d / 2 - a.half);

  // ---- copies: the next group's token, place, and this lane's row of it
  const uint32_t slot0 =
      static_cast<uint32_t>(__cvta_generic_to_shared(&s_rows[warp][0][0][lane]));
  int ct = first, cg = first_group, cg_end = first_group, crow = 0, cheads = 0, to_copy = run;
  const __nv_bfloat16* csrc = nullptr;
  int64_t cstep = 0;
  auto copy = [&](int stage) {
    if (to_copy > 0) {
      --to_copy;
      if (cg == cg_end) {  // a kind of rows begins
        const int from = cg < k_from ? 0 : cg < v_from ? k_from : v_from;
        const int64_t sh = cg < k_from ? a.q_sh : cg < v_from ? a.k_sh : a.v_sh;
        cg_end = cg < k_from ? k_from : cg < v_from ? v_from : all;
        cheads = !there ? 0 : cg < k_from ? a.hq : a.hk;
        crow = (cg - from) * kRows + mine;
        csrc = (cg < k_from ? a.q + ct * a.q_st : cg < v_from ? a.k + ct * a.k_st
                                                              : a.v + ct * a.v_st) + crow * sh;
        cstep = sh * kRows;
      }
      if (crow < cheads) {
        copy16(slot0 + stage * 1024, csrc + lo);
        copy16(slot0 + stage * 1024 + 512, csrc + hi);
      }
      csrc += cstep;
      crow += kRows;
      if (++cg == all) {
        cg = cg_end = 0;
        ++ct;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kDepth; ++i) copy(i);
  int stage = 0;
  auto take = [&](uint4& x, uint4& y) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
    x = s_rows[warp][stage][0][lane];
    y = s_rows[warp][stage][1][lane];
  };
  auto give = [&]() {  // behind the last use of what take() gave
    copy(stage);
    stage = stage + 1 == kDepth ? 0 : stage + 1;
  };

  // ---- this lane's share of a token's angles, and its slot, a token ahead
  const bool angles = kWork && a.half, writes = a.k_pages;
  double freq[kShare], pos[kShare];
  int64_t pos_at[kShare];
#pragma unroll
  for (int x = 0; x < kShare; ++x) {
    freq[x] = pos[x] = 0.;
    pos_at[x] = 0;
    const int i = min(sub * 8 + min(mine * kShare + x, 7), a.half - 1);
    if (angles) {
      freq[x] = static_cast<double>(a.inv_freq[i]) * 0.15915494309189533577;
      pos_at[x] = axis_of(a, i) * a.p_sa;
    }
  }
  int slot = -1;
  auto look = [&](int t) {
    if (t >= a.tokens) return;
    if (angles)
#pragma unroll
      for (int x = 0; x < kShare; ++x) pos[x] = position_at(a, pos_at[x] + t * a.p_st);
    if (writes) slot = a.slots[t];
  };
  look(first);
  const float inv_d = 1.f / static_cast<float>(a.d);

#pragma unroll 1
  for (int t = first, g0 = first_group; run > 0; ++t, g0 = 0) {
    const int g1 = min(all, g0 + run);  // this token's groups
    run -= g1 - g0;
    float mc[kShare], ms[kShare];
    if (kWork && g0 < v_from)
#pragma unroll
      for (int x = 0; x < kShare; ++x) turn(pos[x], freq[x], a.scaling, &mc[x], &ms[x]);
    int64_t page_at = -1;  // where the token's K and V go; -1: nowhere
    if (writes && slot >= 0 && slot < a.num_slots) {
      const int page = slot / a.page_size;
      page_at = page * a.pg_sp + (slot - page * a.page_size) * a.pg_ss;
    } else if (writes && slot != -1 && lane == 0) {
      atomicOr(a.err, UMIC_DEVERR_BAD_PAGE);
    }
    if (run > 0) look(t + 1);

#pragma unroll 1
    for (int kind = g0 < k_from ? 0 : 1; kind < 2; ++kind) {  // q, k
      const int from = kind ? k_from : 0, begin = max(g0, from);
      const int end = min(g1, kind ? v_from : k_from);
      if (begin >= end) continue;
      const bool paged = kind && a.k_pages, e4m3 = kE4m3 && paged;
      int row = (begin - from) * kRows + mine;
      int64_t dst_step = paged ? a.pg_sh : kind ? a.ko_sh : a.qo_sh;
      char* dst = static_cast<char*>(paged ? a.k_pages : kind ? a.k_out : a.q_out);
      dst += ((paged ? page_at : t * (kind ? a.ko_st : a.qo_st)) + row * dst_step) *
             (e4m3 ? 1 : 2);
      dst_step *= e4m3 ? kRows : 2 * kRows;
      const int heads = !there || (paged && page_at < 0) ? 0 : kind ? a.hk : a.hq;  // written
      const void* wt = !kWork ? nullptr : kind ? a.kw : a.qw;
      const float eps = kind ? a.k_eps : a.q_eps;
      // x' = x xc - y ys, y' = y yc + x xs; lanes past the rotated ones: x xc, y yc
      float xc[8], ys[8], yc[8], xs[8];
      if constexpr (kWork) {
#pragma unroll
        for (int i = 0; i < 8; ++i) xc[i] = yc[i] = 1.f;
        if (wt && there) {
          load_w8(wt, a.w_dtype, lo, xc);
          load_w8(wt, a.w_dtype, hi, yc);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int src = min(i / kShare * TPH + sub, 31);
          const float c = __shfl_sync(0xffffffffu, mc[i % kShare], src);
          const float s = __shfl_sync(0xffffffffu, ms[i % kShare], src);
          ys[i] = yc[i] * s;
          xs[i] = xc[i] * s;
          if (turns) {
            xc[i] *= c;
            yc[i] *= c;
          }
        }
      }
#pragma unroll 1
      for (int left = end - begin; left > 0; --left) {
        uint4 xv, yv;
        take(xv, yv);
        if constexpr (!kWork && !kE4m3) {  // as it is
          if (row < heads) {
            st_vec(dst + 2 * lo, xv);
            st_vec(dst + 2 * hi, yv);
          }
          dst += dst_step;
          row += kRows;
          give();
          continue;
        }
        float x[8], y[8];
        unpack8(xv, x);
        unpack8(yv, y);
        float f = 1.f;
        if (wt) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) ss += x[i] * x[i] + y[i] * y[i];
          if (!there || row >= (kind ? a.hk : a.hq)) ss = 0.f;  // pieces not copied
          ss = row_sum<TPH>(ss, mine);
          f = rsqrtf(ss * inv_d + eps);
        }
        if (turns) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float u = x[i] * xc[i] - y[i] * ys[i];
            y[i] = y[i] * yc[i] + x[i] * xs[i];
            x[i] = u;
          }
        } else if (kWork) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] *= xc[i];
            y[i] *= yc[i];
          }
        }
        if (wt) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] *= f;
            y[i] *= f;
          }
        }
        if (row < heads) {
          if (e4m3) {
            if (a.k_scale) divide(x, y, __ldg(a.k_scale + row));
            *reinterpret_cast<uint2*>(dst + lo) = pack8_e4m3(x);
            *reinterpret_cast<uint2*>(dst + hi) = pack8_e4m3(y);
          } else {
            st_vec(dst + 2 * lo, pack8(x));
            st_vec(dst + 2 * hi, pack8(y));
          }
        }
        dst += dst_step;
        row += kRows;
        give();
      }
    }
    // v: a copy, or a rounding to e4m3
    const int begin = max(g0, v_from);
    int row = (begin - v_from) * kRows + mine;
    char* dst = static_cast<char*>(a.v_pages) + (page_at + row * a.pg_sh) * (kE4m3 ? 1 : 2);
    const int heads = there && page_at >= 0 ? a.hk : 0;
#pragma unroll 1
    for (int left = g1 - begin; left > 0; --left) {
      uint4 xv, yv;
      take(xv, yv);
      if (row < heads) {
        if constexpr (kE4m3) {
          float x[8], y[8];
          unpack8(xv, x);
          unpack8(yv, y);
          if (a.v_scale) divide(x, y, __ldg(a.v_scale + row));
          *reinterpret_cast<uint2*>(dst + lo) = pack8_e4m3(x);
          *reinterpret_cast<uint2*>(dst + hi) = pack8_e4m3(y);
        } else {
          st_vec(dst + 2 * lo, xv);
          st_vec(dst + 2 * hi, yv);
        }
      }
      dst += a.pg_sh * (kE4m3 ? kRows : 2 * kRows);
      row += kRows;
      give();
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <int TPH, bool kE4m3>
void launch_work(const MropeArgs& a, bool work, int64_t blocks, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(blocks));
  if (work) launch_pdl(mrope_kernel<TPH, kE4m3, true>, grid, dim3(kThreads), 0, st, a);
  else launch_pdl(mrope_kernel<TPH, kE4m3, false>, grid, dim3(kThreads), 0, st, a);
}
template <int TPH>
void launch(const MropeArgs& a, bool work, int64_t blocks, cudaStream_t st) {
  if (a.e4m3) launch_work<TPH, true>(a, work, blocks, st);
  else launch_work<TPH, false>(a, work, blocks, st);
}

}  // namespace
}  // namespace umic

using namespace umic;

extern "C" int umic_qk_norm_mrope_kv(const umic_mrope_args* args, void* stream) {
  const char* const me = "umic_qk_norm_mrope_kv";
  clear_error();
  if (!args) return fail(UMIC_ERR_INVALID_ARG, "%s: null pointer", me);
  const auto& [q, k, v, q_out, k_out, q_weight, k_weight, positions, inv_freq, k_pages,
               v_pages, k_scale, v_scale, slots, q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st,
               qo_sh, ko_st, ko_sh, p_sa, p_st, pg_sp, pg_sh, pg_ss, num_pages, page_size,
               tokens, hq, hk, head_dim, w_dtype, pos_bytes, rotary_dim, axes, s0, s1, s2,
               interleaved, cache_dtype, q_eps, k_eps, scaling] = *args;
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
  if (tokens > 0x7fff0000LL)
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
  // rows written: apart from one another
  if ((hq > 0 && !rows_apart({{tokens, qo_st}, {hq, qo_sh}}, head_dim)) ||
      !(k_pages ? rows_apart({{num_pages, pg_sp}, {hk, pg_sh}, {page_size, pg_ss}}, head_dim)
                : rows_apart({{tokens, ko_st}, {hk, ko_sh}}, head_dim)))
    return fail(UMIC_ERR_INVALID_ARG, "%s: output rows overlap", me);
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
  // Lanes of a row: a power of two, but for the 5 and 6 that head_dim 80 and 96 fill. 16384
  // tokens of 16 + 16 heads x 80, two axes: 37.5 us with 5 lanes, 38.7 with 8; normed, three
  // axes, 16 + 8 + 8 heads into pages 43.5 and 46.0, written as they are 38.4 and 36.5. x 96:
  // 38.4 with 6 lanes, 39.2 with 8; 47.0 and 46.9; 40.1 and 39.8. Other sizes keep idle lanes:
  // no model here has them.
  const int tph = head_dim <= 64 ? 4 : head_dim == 80 ? 5 : head_dim == 96 ? 6
                  : head_dim <= 128 ? 8 : 16;
  const int at_once = 32 / tph;
  const bool work = rotary_dim > 0 || q_weight || k_weight;
  const int per_sm = blocks_per_sm(work);
  const int64_t groups = (static_cast<int64_t>(hq) + at_once - 1) / at_once +
                         (static_cast<int64_t>(hk) + at_once - 1) / at_once * (k_pages ? 2 : 1);
  if (groups > (1 << 20))
    return fail(UMIC_ERR_UNSUPPORTED, "%s: too many heads (%d + %d)", me, hq, hk);
  // a group for every resident warp, more while there are more
  const int64_t total = tokens * groups;
  const int64_t blocks = std::min<int64_t>((total + kThreads / 32 - 1) / (kThreads / 32),
                                           static_cast<int64_t>(sm_count()) * per_sm);
  const int64_t warps = blocks * (kThreads / 32);
  a.run = total / warps;
  a.longer = static_cast<int32_t>(total % warps);
  if (a.run >= 0x7fffffffLL)
    return fail(UMIC_ERR_UNSUPPORTED, "%s: %lld tokens x %lld heads", me, (long long)tokens,
                (long long)hq + hk);
  cudaStream_t st = as_stream(stream);
  if (tph == 4) launch<4>(a, work, blocks, st);
  else if (tph == 5) launch<5>(a, work, blocks, st);
  else if (tph == 6) launch<6>(a, work, blocks, st);
  else if (tph == 8) launch<8>(a, work, blocks, st);
  else launch<16>(a, work, blocks, st);
  return launch_status(me);
}
