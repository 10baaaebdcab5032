// Block tables and the slot map of one serving step, built on the device from request
// lengths (umic_paged_plan).
//
// Every request's share is a prefix sum over the requests before it: the pages it takes
// from the ring of free pages, the pages it gives back, and the place of its tokens among
// the step's. What there is to read and write is small (8 bytes a token of the step), so
// the chain of dependent steps bounds it: read the lengths, scan, write. One cluster of up
// to 8 CTAs does it in one launch. Every CTA scans all requests (a run of them per thread)
// and keeps in shared memory where each one's tokens and pages begin; then each takes its
// part of the pages that change hands, a warp a request, and of the tokens, which find
// their request by binary search. out_lens and out_span may lie over the inputs: they are
// written behind a cluster barrier that every CTA reaches with its reading done. Measured:
// 8 requests of one token 5.5 us, 1024 (a tenth of them ending) 10.3 us, 99200 prompt
// tokens of 32 requests 10.1 us.
#include "common.cuh"

namespace umic {
namespace {

constexpr int kMostThreads = 1024;
constexpr int64_t kMaxRequests = 8192;
constexpr int kMostEach = kMaxRequests / kMostThreads;  // requests a thread scans, at most
// Pages of a request that the scanning thread moves itself. Requests that take two or three
// gain by it (64, 512 and 1024 prompts of 32 tokens on pages of 16: 6.6, 9.4 and 10.5 us,
// against 6.9, 10.3 and 11.2 with one), steps of one token lose 0.2 us; with 16 all lose 1 to
// 1.5 us.
constexpr int kFew = 4;

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
  int64_t table_stride, num_pages, capacity;
  int32_t max_tokens;  // of a row
  int32_t requests, page_size;
  bool wide;  // slots and positions take 16-byte stores
};

// What a request asks for. A length is valid if it fits its row, so pages are 32-bit.
struct Ask {
  int32_t len, change;    // length before, tokens appended or (negative) dropped
  int32_t before, after;  // pages
  bool valid;
};

__device__ __forceinline__ Ask ask_of(const PlanArgs& a, int r) {
  Ask q;
  q.len = a.lens[r];
  q.change = a.delta[r];
  const int64_t then = static_cast<int64_t>(q.len) + q.change;
  q.valid = q.len >= 0 && q.len <= a.max_tokens && then >= 0 && then <= a.max_tokens;
  if (!q.valid) q.change = 0;
  const uint32_t page = a.page_size;
  q.before = q.valid ? static_cast<uint32_t>(q.len) / page : 0;
  q.after = q.valid ? static_cast<uint32_t>(then) / page : 0;
  if (q.valid) {  // rounded up
    q.before += static_cast<uint32_t>(q.len) - q.before * page != 0;
    q.after += static_cast<uint32_t>(then) - q.after * page != 0;
  }
  return q;
}

// Pages taken, pages given back, tokens appended, each held at 2^31 - 1: what is past it is
// past the free pages and the capacity too, and a sum that stops there can be taken in any
// grouping. (64-bit sums double the shuffles of the scan.)
__device__ __forceinline__ uint32_t capped(uint32_t x, uint32_t y) {
  return min(x + y, 0x7fffffffu);
}
struct Sums {
  uint32_t need, give, count;
  __device__ Sums plus(const Sums& o) const {
    return {capped(need, o.need), capped(give, o.give), capped(count, o.count)};
  }
};
__device__ __forceinline__ Sums sums_of(const Ask& q) {
  return {static_cast<uint32_t>(max(q.after - q.before, 0)),
          static_cast<uint32_t>(max(q.before - q.after, 0)),
          static_cast<uint32_t>(max(q.change, 0))};
}
__device__ __forceinline__ Sums from_lane(const Sums& s, int lane) {
  return {__shfl_sync(0xffffffffu, s.need, lane), __shfl_sync(0xffffffffu, s.give, lane),
          __shfl_sync(0xffffffffu, s.count, lane)};
}
__device__ __forceinline__ Sums warp_scan(Sums s, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Sums left = from_lane(s, max(lane - o, 0));
    if (lane >= o) s = s.plus(left);
  }
  return s;
}

// Sums of the threads before this one; the block's in *total.
__device__ __forceinline__ Sums block_scan(const Sums& mine, Sums* total) {
  __shared__ Sums warp_sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const Sums inc = warp_scan(mine, lane);
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  const Sums all = warp_scan(lane < warps ? warp_sums[lane] : Sums{0, 0, 0}, lane);
  *total = from_lane(all, 31);
  const Sums before = from_lane(inc, max(lane - 1, 0)), base = from_lane(all, max(warp - 1, 0));
  const Sums zero{0, 0, 0};
  return (warp > 0 ? base : zero).plus(lane > 0 ? before : zero);
}

// i modulo n for 0 <= i < 2 n
__device__ __forceinline__ int32_t fold(int64_t i, int64_t n) {
  return static_cast<int32_t>(i >= n ? i - n : i);
}
// i modulo n, for any i
__device__ __forceinline__ int64_t modulo(int64_t i, int64_t n) {
  if (i >= 0 && i <= 0xffffffffLL) return static_cast<uint32_t>(i) % static_cast<uint32_t>(n);
  i %= n;
  return i < 0 ? i + n : i;
}

__global__ void __launch_bounds__(kMostThreads) paged_plan_kernel(PlanArgs a) {
  // per request: its first token of the step; its length before, or -1: not served; pages
  // before; ring place of its first new (or returned) page. Then pages after.
  extern __shared__ int4 s_place[];
  int32_t* const s_after = reinterpret_cast<int32_t*>(s_place + a.requests);
  __shared__ uint32_t s_taken;
  const int ctas = gridDim.x, cta = blockIdx.x;  // the grid is one cluster
  const int threads = blockDim.x, lane = threadIdx.x & 31;
  allow_dependent_launch();
  if (threadIdx.x == 0) s_taken = 0;
  wait_prerequisite();
  const int64_t head = a.span[0], tail = a.span[1];

  const int per = (a.requests + threads - 1) / threads;
  const int r0 = min(a.requests, static_cast<int>(threadIdx.x) * per);
  const int r1 = min(a.requests, r0 + per);
  Sums mine{0, 0, 0};
  Ask kept{};  // the only one, mostly: read once
  for (int r = r0; r < r1; ++r) {
    kept = ask_of(a, r);
    mine = mine.plus(sums_of(kept));
  }
  Sums total;
  Sums at = block_scan(mine, &total);
  const int64_t free_pages = max(int64_t{0}, min(tail - head, a.num_pages));
  const int64_t tokens = total.count, head_mod = modulo(head, a.num_pages);
  const int64_t tail_mod = modulo(tail, a.num_pages);
  bool refused = false;
  for (int r = r0; r < r1; ++r) {
    const Ask q = per == 1 ? kept : ask_of(a, r);
    const int need = max(q.after - q.before, 0), give = max(q.before - q.after, 0);
    const bool served =
        q.valid && (need == 0 || static_cast<int64_t>(at.need) + need <= free_pages) &&
        (q.change <= 0 || static_cast<int64_t>(at.count) + q.change <= a.capacity);
    refused |= !served;
    // a served request's pages lie within one turn of the ring behind head, returned ones
    // within the pool's pages behind tail
    const int32_t place = need ? (served ? fold(head_mod + at.need, a.num_pages) : 0)
                               : static_cast<int32_t>(modulo(tail_mod + at.give, a.num_pages));
    s_place[r] = make_int4(at.count, served ? q.len : -1, q.before, place);
    s_after[r] = served ? q.after : q.before;
    // the requests that take pages and are served are a prefix of those that ask for
    // pages, so the pages taken are the largest end among them
    if (served && need) atomicMax(&s_taken, at.need + need);
    if (served && need + give <= kFew && r % ctas == cta) {
      int32_t* const row = a.table + r * a.table_stride;
      int32_t moved[kFew];
#pragma unroll
      for (int j = 0; j < kFew; ++j)
        if (j < need) moved[j] = a.ring[fold(static_cast<int64_t>(place) + j, a.num_pages)];
        else if (j < give) moved[j] = row[q.after + j];
#pragma unroll
      for (int j = 0; j < kFew; ++j)
        if (j < need) row[q.before + j] = moved[j];
        else if (j < give) a.ring[modulo(static_cast<int64_t>(place) + j, a.num_pages)] = moved[j];
    }
    at = at.plus(sums_of(q));
  }
  if (refused && cta == 0) atomicOr(a.err, UMIC_DEVERR_PAGES);
  __syncthreads();

  // ---- more pages that change hands, a warp a request: new ones out of the ring, and given
  // back to its end (never where pages are taken: the ring holds every page of the pool)
  for (int r = cta + ctas * static_cast<int>(threadIdx.x >> 5); r < a.requests;
       r += ctas * (threads >> 5)) {
    const int4 p = s_place[r];
    const int after = s_after[r];
    if (abs(after - p.z) <= kFew) continue;
    int32_t* const row = a.table + r * a.table_stride;
    for (int j = p.z + lane; j < after; j += 32)
      row[j] = a.ring[fold(static_cast<int64_t>(p.w) + j - p.z, a.num_pages)];
    for (int j = after + lane; j < p.z; j += 32)
      a.ring[modulo(static_cast<int64_t>(p.w) + j - after, a.num_pages)] = row[j];
  }

  // ---- tokens, four a thread
  const int64_t quads = (a.capacity + 3) / 4;
  bool bad = false;
  for (int64_t i = static_cast<int64_t>(cta) * threads + threadIdx.x; i < quads;
       i += static_cast<int64_t>(ctas) * threads) {
    int32_t slot[4], pos[4];
    int r = -1, next_start = 0;
    int32_t n_last = -1, page = -1;
    int4 p = make_int4(0, -1, 0, 0);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t t = 4 * i + u;
      slot[u] = pos[u] = -1;
      if (t >= tokens || t >= a.capacity) continue;
      if (t >= next_start) {  // the last request that begins at or before t
        int lo = max(r, 0), hi = a.requests;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (s_place[mid].x <= t) lo = mid; else hi = mid;
        }
        r = lo;
        p = s_place[r];
        next_start = r + 1 < a.requests ? s_place[r + 1].x : 0x7fffffff;
        n_last = -1;
      }
      if (p.y < 0) continue;
      const int32_t at_pos = p.y + static_cast<int32_t>(t - p.x);
      const int32_t n = static_cast<uint32_t>(at_pos) / static_cast<uint32_t>(a.page_size);
      if (n != n_last) {
        n_last = n;
        page = n >= p.z ? a.ring[fold(static_cast<int64_t>(p.w) + n - p.z, a.num_pages)]
                        : a.table[r * a.table_stride + n];
      }
      if (page < 0 || page >= a.num_pages) {
        bad = true;
      } else {
        slot[u] = page * a.page_size + (at_pos - n * a.page_size);
        pos[u] = at_pos;
      }
    }
    if (a.wide && 4 * i + 4 <= a.capacity) {
      *reinterpret_cast<int4*>(a.slots + 4 * i) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *reinterpret_cast<int4*>(a.positions + 4 * i) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (4 * i + u < a.capacity) {
          a.slots[4 * i + u] = slot[u];
          a.positions[4 * i + u] = pos[u];
        }
    }
  }
  if (bad) atomicOr(a.err, UMIC_DEVERR_BAD_PAGE);

  // ---- what may lie over the inputs: the lengths and the span, behind every CTA's reading.
  // A request that is not served keeps its length, which is read once more.
  int32_t lens[kMostEach];
  int n = 0;
  for (int r = cta * threads + threadIdx.x; r < a.requests; r += ctas * threads, ++n)
    lens[n] = s_place[r].y < 0 ? a.lens[r] : s_place[r].y + a.delta[r];
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
  n = 0;
  for (int r = cta * threads + threadIdx.x; r < a.requests; r += ctas * threads, ++n) {
    a.out_lens[r] = lens[n];
    a.cu[r] = s_place[r].x;
  }
  if (cta == 0 && threadIdx.x == 0) {
    a.cu[a.requests] = total.count;
    a.out_span[0] = head + s_taken;
    a.out_span[1] = tail + total.give;
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
  const bool wide =
      ((reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(positions)) & 15u) == 0;
  PlanArgs a{kv_lens,   new_tokens, block_table,  free_ring, free_span,
             out_lens,  out_span,   cu_tokens,    slots,     positions,
             err,       table_stride, num_pages,  capacity,
             static_cast<int32_t>(max_pages * page_size),
             static_cast<int32_t>(requests), static_cast<int32_t>(page_size), wide};
  const size_t smem = static_cast<size_t>(requests) * (sizeof(int4) + sizeof(int32_t));
  static std::once_flag once[64];
  int dev = 0;
  cudaGetDevice(&dev);
  std::call_once(once[dev & 63], [] {
    cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         static_cast<int>(kMaxRequests * (sizeof(int4) + sizeof(int32_t))));
  });
  // One small CTA while four tokens a thread and a request a thread cover the step and its
  // four warps hide their look-ups: against 1024 threads, 8 requests of one token take 5.4 us
  // to 6.0, 32 take 6.45 to 6.65, 48 take 6.9 to 6.85, 128 take 9.1 to 7.6, and one prompt of
  // 512 tokens 3.8 to 4.5. Else large ones, twice as many while there are more than 4096
  // tokens or 128 requests for each: 1, 2, 4 and 8 CTAs take 12.5, 11.3, 10.5 and 10.2 us for
  // 1024 requests, 15.4 to 10.3 with a tenth of them ending, 8.5, 7.0, 5.7 and 5.8 for four
  // prompts of 3100 tokens, 42, 24, 14 and 10 for 32.
  const int threads = requests <= 40 && capacity <= 512 ? 128 : kMostThreads;
  int ctas = 1;
  while (threads == kMostThreads && ctas < 8 && (capacity > 4096 * ctas || requests > 128 * ctas))
    ctas *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = as_stream(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, paged_plan_kernel, a);
  return launch_status("umic_paged_plan");
}
