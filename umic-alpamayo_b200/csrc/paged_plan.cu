// Block tables and the slot map of one serving step, built on the device from request
// lengths (umic_paged_plan).
//
// Every request's share is a prefix sum over the requests before it: the pages it
// takes from the ring of free pages, the pages it gives back, and the place of its
// tokens among the step's. One CTA scans the three sums (a run of consecutive requests
// per thread), keeps per request where its tokens and pages begin in shared memory,
// and then walks the pages that change hands and the step's tokens; a token finds its
// request by binary search over the token offsets.
#include "common.cuh"

namespace umic {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int64_t kMaxRequests = 8192;

struct PlanArgs {
  const int32_t* lens;
  const int32_t* delta;
  int32_t* table;
  int32_t* ring;
  const int64_t* span;
  int32_t* out_lens;
  int64_t* out_span;
  int32_t* cu;
  int32_t* slots;
  int32_t* positions;
  uint32_t* err;
  int64_t table_stride, max_pages, num_pages, capacity;
  int32_t requests, page_size;
};

struct Ask {
  int64_t old_len, new_len;  // lengths before and after, were it served
  int64_t before, after;     // pages before and after
  bool valid;
  __device__ int64_t need() const { return after > before ? after - before : 0; }
  __device__ int64_t give() const { return before > after ? before - after : 0; }
  __device__ int64_t count() const { return new_len > old_len ? new_len - old_len : 0; }
};

__device__ __forceinline__ Ask ask_of(const PlanArgs& a, int r) {
  Ask q;
  q.old_len = a.lens[r];
  q.new_len = q.old_len + a.delta[r];
  q.valid = q.old_len >= 0 && q.new_len >= 0;
  q.before = q.valid ? (q.old_len + a.page_size - 1) / a.page_size : 0;
  q.after = q.valid ? (q.new_len + a.page_size - 1) / a.page_size : 0;
  if (q.before > a.max_pages || q.after > a.max_pages) q.valid = false;
  if (!q.valid) {
    q.new_len = q.old_len;
    q.after = q.before;
  }
  return q;
}

struct Sums {
  int64_t need, give, count;
};

// Exclusive sums over the threads before this one; the block's totals in `total`.
__device__ Sums block_scan(Sums mine, Sums* total) {
  __shared__ Sums warp_sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Sums inc = mine;
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t n = __shfl_up_sync(0xffffffffu, inc.need, o);
    const int64_t g = __shfl_up_sync(0xffffffffu, inc.give, o);
    const int64_t c = __shfl_up_sync(0xffffffffu, inc.count, o);
    if (lane >= o) {
      inc.need += n;
      inc.give += g;
      inc.count += c;
    }
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  Sums base{0, 0, 0}, all{0, 0, 0};
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) {
    if (w == warp) base = all;
    all.need += warp_sums[w].need;
    all.give += warp_sums[w].give;
    all.count += warp_sums[w].count;
  }
  *total = all;
  return {base.need + inc.need - mine.need, base.give + inc.give - mine.give,
          base.count + inc.count - mine.count};
}

__device__ __forceinline__ int32_t clamp31(int64_t x) {
  return static_cast<int32_t>(x > 0x7fffffffLL ? 0x7fffffffLL : x);
}

// (base + i) modulo num_pages, for any base
__device__ __forceinline__ int64_t wrap(int64_t i, int64_t n) {
  i %= n;
  return i < 0 ? i + n : i;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PlanArgs a) {
  // per request: first token of the step, length before (-1: not served), pages before,
  // ring place of its first new page
  extern __shared__ int32_t sh[];
  int32_t* s_start = sh;
  int32_t* s_len = sh + a.requests;
  int32_t* s_before = sh + 2 * a.requests;
  int32_t* s_take = sh + 3 * a.requests;
  __shared__ int64_t s_given_end;

  allow_dependent_launch();
  wait_prerequisite();
  const int64_t head = a.span[0], tail = a.span[1];
  int64_t free_pages = tail - head;
  free_pages = free_pages < 0 ? 0 : free_pages > a.num_pages ? a.num_pages : free_pages;

  const int per = (a.requests + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min(a.requests, static_cast<int>(threadIdx.x) * per);
  const int r1 = min(a.requests, r0 + per);
  Sums mine{0, 0, 0};
  for (int r = r0; r < r1; ++r) {
    const Ask q = ask_of(a, r);
    mine.need += q.need();
    mine.give += q.give();
    mine.count += q.count();
  }
  Sums total;
  Sums at = block_scan(mine, &total);
  const int64_t tokens = total.count;
  if (threadIdx.x == 0) {
    s_given_end = tail + total.give;
    a.cu[a.requests] = clamp31(tokens);
  }
  // the requests that take pages and are served are a prefix of those that ask for
  // pages, so the pages taken are the largest end among them
  __shared__ unsigned long long s_taken;
  if (threadIdx.x == 0) s_taken = 0;
  __syncthreads();
  bool refused = false;
  for (int r = r0; r < r1; ++r) {
    const Ask q = ask_of(a, r);
    const int64_t need = q.need(), count = q.count();
    const bool served = q.valid && (need == 0 || at.need + need <= free_pages) &&
                        (count == 0 || at.count + count <= a.capacity);
    refused |= !served;
    s_start[r] = clamp31(at.count);
    a.cu[r] = s_start[r];
    s_len[r] = served ? static_cast<int32_t>(q.old_len) : -1;
    s_before[r] = static_cast<int32_t>(q.before);
    s_take[r] = static_cast<int32_t>(wrap(head + at.need, a.num_pages));
    if (served && need) atomicMax(&s_taken, static_cast<unsigned long long>(at.need + need));
    // pages given back go to the end of the ring (never where pages are taken: the
    // ring holds every page of the pool)
    if (served) {
      for (int64_t j = q.after; j < q.before; ++j)
        a.ring[wrap(tail + at.give + j - q.after, a.num_pages)] = a.table[r * a.table_stride + j];
      for (int64_t j = q.before; j < q.after; ++j)
        a.table[r * a.table_stride + j] =
            a.ring[wrap(head + at.need + j - q.before, a.num_pages)];
      a.out_lens[r] = static_cast<int32_t>(q.new_len);
    } else {
      a.out_lens[r] = a.lens[r];
    }
    at.need += need;
    at.give += q.give();
    at.count += count;
  }
  if (refused) atomicOr(a.err, UMIC_DEVERR_PAGES);
  __syncthreads();
  if (threadIdx.x == 0) {
    a.out_span[0] = head + static_cast<int64_t>(s_taken);
    a.out_span[1] = s_given_end;
  }
  for (int64_t t = threadIdx.x; t < a.capacity; t += blockDim.x) {
    int32_t slot = -1, pos = -1;
    if (t < tokens) {
      int lo = 0, hi = a.requests;  // the last request that begins at or before t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_start[mid] <= t) lo = mid; else hi = mid;
      }
      if (s_len[lo] >= 0) {
        pos = s_len[lo] + static_cast<int32_t>(t - s_start[lo]);
        const int32_t i = pos / a.page_size;
        const int32_t page =
            i >= s_before[lo]
                ? a.ring[wrap(static_cast<int64_t>(s_take[lo]) + i - s_before[lo], a.num_pages)]
                : a.table[lo * a.table_stride + i];
        if (page < 0 || page >= a.num_pages) {
          slot = pos = -1;
          atomicOr(a.err, UMIC_DEVERR_BAD_PAGE);
        } else {
          slot = page * a.page_size + pos % a.page_size;
        }
      }
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
  }
}

}  // namespace
}  // namespace umic

using namespace umic;

extern "C" int umic_paged_plan(const int32_t* kv_lens, const int32_t* new_tokens,
                               int64_t requests, int32_t* block_table, int64_t table_stride,
                               int64_t max_pages, int32_t* free_ring, int64_t num_pages,
                               const int64_t* free_span, int64_t page_size, int32_t* out_lens,
                               int64_t* out_span, int32_t* cu_tokens, int32_t* slots,
                               int32_t* positions, int64_t capacity, void* stream) {
  clear_error();
  if (requests <= 0 || max_pages <= 0 || num_pages <= 0 || page_size <= 0 || capacity < 0)
    return fail(UMIC_ERR_INVALID_ARG,
                "umic_paged_plan: requests=%lld max_pages=%lld num_pages=%lld page_size=%lld "
                "capacity=%lld",
                (long long)requests, (long long)max_pages, (long long)num_pages,
                (long long)page_size, (long long)capacity);
  if (!kv_lens || !new_tokens || !block_table || !free_ring || !free_span || !out_lens ||
      !out_span || !cu_tokens || (capacity > 0 && (!slots || !positions)))
    return fail(UMIC_ERR_INVALID_ARG, "umic_paged_plan: null pointer");
  if (requests > 1 && table_stride < max_pages)
    return fail(UMIC_ERR_INVALID_ARG, "umic_paged_plan: table rows overlap (stride %lld < %lld)",
                (long long)table_stride, (long long)max_pages);
  if (requests > kMaxRequests)
    return fail(UMIC_ERR_UNSUPPORTED, "umic_paged_plan: %lld requests (at most %lld)",
                (long long)requests, (long long)kMaxRequests);
  if (page_size > 0x7fffffffLL / num_pages || page_size > 0x7fffffffLL / max_pages ||
      capacity > 0x7fffffffLL)
    return fail(UMIC_ERR_UNSUPPORTED,
                "umic_paged_plan: num_pages * page_size, max_pages * page_size and capacity "
                "must stay below 2^31");
  if ((reinterpret_cast<uintptr_t>(free_span) | reinterpret_cast<uintptr_t>(out_span)) & 7u)
    return fail(UMIC_ERR_ALIGNMENT, "umic_paged_plan: free_span / out_span not 8-byte aligned");
  uint32_t* err = device_error_word();
  if (!err) return fail(UMIC_ERR_DEVICE, "umic_paged_plan: no device error word");
  PlanArgs a{kv_lens,      new_tokens, block_table, free_ring, free_span,
             out_lens,     out_span,   cu_tokens,   slots,     positions,
             err,          table_stride, max_pages, num_pages, capacity,
             static_cast<int32_t>(requests), static_cast<int32_t>(page_size)};
  const size_t smem = static_cast<size_t>(requests) * 16;
  static std::once_flag once[64];
  int dev = 0;
  cudaGetDevice(&dev);
  std::call_once(once[dev & 63], [] {
    cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         static_cast<int>(kMaxRequests) * 16);
  });
  launch_pdl(paged_plan_kernel, dim3(1), dim3(kPlanThreads), smem, as_stream(stream), a);
  return launch_status("umic_paged_plan");
}
