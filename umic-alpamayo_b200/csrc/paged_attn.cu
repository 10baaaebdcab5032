// Attention of one new token per request over its key-value pages (umic_paged_attention).
//
//   out[b, h] = sum_j softmax_j(scale q[b, h] . k_j) v_j,  j < kv_lens[b]
//
// Every K and V byte is used once, for the G query heads of its KV head: 2 G flops a byte
// (bf16) against the hundreds that the tensor cores could do, so HBM bounds the kernel and
// all that matters is to keep its loads in flight.
//
// Work. A segment is one request's one KV head (up to 8 * NT query heads; wider groups are
// cut into several segments), a tile 16 or 32 of its tokens. All tiles of all segments form
// one line, and every warp takes an equal run of it, whatever the lengths: no warp idles
// because its request is short. A warp needs no other: it copies its tiles into its own
// ring with 16-byte asynchronous loads, kStages ahead across segment borders, and waits for
// its own copies only. (Runs that warps claim from a counter as they come free, to even out
// the SMs' shares of HBM, cost more in partial results than they gained.) Per tile:
//   S^T = K Q^T    mma.sync m16n8k16, tokens as rows: the 8 columns are query heads, so a
//                  group of up to 8 heads costs one instruction per 16 dims (tcgen05 wants
//                  64 or 128 rows per operand and a block-wide hand-over of each tile;
//                  here the tensor pipe is busy 10 to 16 per cent of the time)
//   m, l, P        running maximum and sum of each head, fp32, base 2
//   O^T += V^T P   V through transposing ldmatrix, P transposed in registers
// P is fp32 split into a bf16 value and its bf16 remainder (two products, weights held to
// 2^-17): the tensor pipe has the time. (Where V is infinite a remainder of 0 makes NaN.)
// e4m3 pages are widened to fp16 in registers, which holds them exactly. q is scaled by the
// power of two of its row's largest to stay inside fp16: what is below 2^-14 of that is held
// to 2^-25 of it. P is held as one fp16 value times 2^15, so that small weights stay normal:
// each is off by 2^-11 of itself at most, while their sum takes them unrounded. Two fp16
// terms, as for bf16 pages, took 220 us for 205 (256 requests of up to 4096 tokens, 16 and 8
// heads) and left the error against 64 bits, 0.0017 of the outputs' size by their own
// rounding to bf16, as it was. (The e4m3 form of mma.sync is made of conversions and fp16
// products here: more instructions, not fewer.)
//
// Join. A warp whose run covers a whole segment writes its rows. Otherwise it has partial
// (m, l, O): neighbours of one CTA that share a segment join through shared memory, and
// what still crosses CTAs goes to the workspace, where a second kernel joins the partials
// of each split segment in line order. Sums are taken in a fixed order: results repeat bit
// for bit. (The last CTA of a segment joining it, in one kernel, took 5 us more: code that
// runs once, at the end, from a cold instruction cache.)
//
// Measured, both kernels, 32 query and 8 KV heads x 128: 32 requests of up to 32768 tokens
// (2.2 GB) 348 us, 0.96 of measured HBM; 8 of 3164 tokens (104 MB) 26.6 us, of which 16 us
// stream and 10 us are start, join and the spread of the warps' ends; 1 of 3164 12.9 us.
// 256 requests of up to 4096 tokens in e4m3 pages, 16 and 8 heads (1.04 GB) 205 us: there
// the widening (half of a tile's instructions) bounds it as much as HBM. 128 requests of up
// to 4096 tokens, two query heads to a KV head, 16 KV heads of 64, 80, 96, 128 (8 of 256), in
// bf16: 187, 243, 283, 346, 343 us, 0.81 to 0.91; in e4m3: 154, 172, 191, 217, 222 us, 0.51 to
// 0.72. 256 of up to 4096, 4 KV heads x 128: 16 query heads to each 200 us (0.79), e4m3 167
// (0.48); 32 to each, whose two segments read K and V twice, 348 (0.46) and 303 (0.27).
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"

namespace umic {
namespace {

constexpr int kSub = 16;              // tokens per subtile: rows of one mma, within one page
constexpr float kF16Shift = 15.f;     // e4m3 path: weights are held as 2^15 p
constexpr int kSmemBudget = 216 * 1024;

// A split segment, left by the run that holds its first tile for the joining kernel.
struct Split {
  int32_t b;     // request, or -1: none begins here
  int32_t hc;    // segment of the request
  int32_t last;  // run that holds its last tile
  int32_t head;  // 1: that run goes on behind the segment
};

// The workspace: the splits, and two partial results for each warp's run (0: of its last
// segment, 1: of its first if that is another).
struct Space {
  char* base;
  int64_t runs;  // room for
  __host__ __device__ Split* splits() const { return reinterpret_cast<Split*>(base); }
  __host__ __device__ float* slot(int64_t run, int head, int floats) const {
    return reinterpret_cast<float*>(splits() + runs) + (run * 2 + head) * floats;
  }
  static constexpr size_t bytes(int64_t runs, int64_t floats) {
    return runs * (sizeof(Split) + 2 * floats * sizeof(float));
  }
};

struct PagedArgs {
  const __nv_bfloat16* q;
  const char *k_pages, *v_pages;
  const float *k_scale, *v_scale;
  const int32_t *table, *lens;
  __nv_bfloat16* out;
  float* lse;
  uint32_t* err;
  Space ws;
  int64_t q_sb, q_sh, pg_sp, pg_sh, pg_ss;  // pg_* in bytes
  int64_t table_stride, num_pages, o_sb, o_sh;
  int32_t max_len, max_pages, page_size, hq, hkv, batch, group, chunks;  // chunks: segments per KV head
  float scale_log2;
};

// Subtiles of a tile: two for rows of up to 192 bytes, whose running maximum and shuffles
// cost a tile the same whatever it holds (the cases of two query heads above with one: bf16
// 200, 256, 298 us for head dims 64, 80, 96; e4m3 192, 212, 226, 254 for 64 to 128). Two of
// rows of 256 bytes, 16 KB of K and V, would leave eight warps one stage.
constexpr int subtiles(int d, bool e4m3) { return d * (e4m3 ? 1 : 2) <= 192 ? 2 : 1; }
// Warps of a CTA. bf16: 8, of whose ring of three 8 KB tiles two fill while one is used
// (head_dim 256: 4, whose 16 KB tiles and accumulators fit). e4m3: the work of widening,
// twice per byte, wants 12 to hide its latencies (the cases of two query heads above, head
// dims 64 to 256: 154, 172, 191, 217, 222 us, against 194, 196, 212, 248, 227 with 8; 16
// query heads x 64: 185 against 216), unless two column tiles' accumulators leave room for 8
// only.
constexpr int warps_per_cta(int d, bool e4m3, int per) {
  return e4m3 ? (d >= 128 && per > 8 ? 8 : 12) : d == 256 ? 4 : 8;
}

// Shapes of one instantiation.
template <int D, bool kE4m3, int NT>
struct Shape {
  static constexpr int kRow = D * (kE4m3 ? 1 : 2);                   // bytes of a token's row
  // Rows in shared memory, so that eight rows' same 16 bytes fall in different banks: whole
  // 128-byte lines with their 16-byte pieces exchanged (piece p of row r at p ^ r % 8), else
  // padded to an odd count of pieces. (Padding 256-byte rows too was 6 per cent slower:
  // copies then straddle lines.)
  static constexpr bool kSwizzle = kRow % 128 == 0;
  static constexpr int kPitch = kSwizzle ? kRow : kRow + ((kRow / 16) % 2 ? 0 : 16);
  __device__ static uint32_t piece(int row, int p) {
    return row * kPitch + (kSwizzle ? p ^ (row & 7) : p) * 16;
  }
  // the piece `bytes` further on in a row, from one whose number has those bits clear
  __device__ static uint32_t along(uint32_t at, int bytes) {
    return kSwizzle ? at ^ bytes : at + bytes;
  }
  static constexpr int MT = subtiles(D, kE4m3);
  static constexpr int kTile = kSub * MT;                           // tokens per tile
  static constexpr int kSubBytes = 2 * kSub * kPitch;               // K, then V
  static constexpr int kTileBytes = MT * kSubBytes;
  static constexpr int kWarps = warps_per_cta(D, kE4m3, 8 * NT);
  static constexpr int kFit = kSmemBudget / (kWarps * kTileBytes);
  static constexpr int kStages = kFit < 6 ? kFit : 6;
  static constexpr int kBlocks = D / 16;                            // 16-dim blocks
  static constexpr int kOut = NT * kBlocks * 128;                   // floats of one partial O
  static constexpr int kSlot = kOut + NT * 16;                      // + m and l of 8 * NT heads
  static constexpr size_t kSmem = static_cast<size_t>(kWarps) * kStages * kTileBytes + 512;
  static_assert(kStages >= 2, "one tile in use, one in flight");
  static_assert(kStages * kTileBytes >= kSlot * 4, "a partial result fits its warp's ring");
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm2(uint32_t& r0, uint32_t& r1, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];"
               : "=r"(r0), "=r"(r1)
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm2t(uint32_t& r0, uint32_t& r1, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];"
               : "=r"(r0), "=r"(r1)
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// Not volatile: products of different accumulators may be moved past one another, so that
// a chain's next product need not wait for the last.
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Four e4m3 values as fp16 pairs (bytes 0, 2 and bytes 1, 3), times kWide, exactly. The
// seven bits below the sign, put three places higher in fp16, are the value times 2^-8,
// subnormals included; the product with 2^8 kWide has 4 + 6 bits, is normal, and sends the
// NaN code (which the shift makes 480 * 2^-8) over the largest fp16 to infinity, which the
// scores and the output turn into NaN again. Nine instructions, five of them on the ALU pipe,
// which the conversion instruction would fill.
constexpr float kWide = 140.f;
__device__ __forceinline__ void widen4(uint32_t r, uint32_t& even, uint32_t& odd) {
  const uint32_t e = ((r * 256u) & 0x80008000u) | ((r * 128u) & 0x3f803f80u);
  const uint32_t o = (r & 0x80008000u) | ((r >> 1) & 0x3f803f80u);
  const __half2 up = __float2half2_rn(256.f * kWide);
  const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&e), up);
  const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&o), up);
  even = *reinterpret_cast<const uint32_t*>(&x);
  odd = *reinterpret_cast<const uint32_t*>(&y);
}

__device__ __forceinline__ int clamped_len(const PagedArgs& a, int b) {
  return max(0, min(a.lens[b], a.max_len));
}

// The line of `total` tiles cut into `workers` runs, the first `longer` one tile longer.
// (32-bit: a 64-bit division takes hundreds of cycles here.)
struct Line {
  int base, longer;
  __device__ Line(int total, int workers) : base(total / workers), longer(total % workers) {}
  __device__ int begin(int w) const { return w * base + min(w, longer); }
  __device__ int run_of(int x) const {
    const int cut = longer * (base + 1);
    return x < cut ? x / (base + 1) : longer + (x - cut) / base;
  }
};

// One warp's view of a segment's rows: where the outputs of its heads go.
template <int D, bool kE4m3, int NT>
struct Rows {
  __device__ static int head0(const PagedArgs& a, int hc) {  // first query head of a segment
    return hc / a.chunks * a.group + hc % a.chunks * (8 * NT);
  }
  __device__ static int heads(const PagedArgs& a, int hc) {
    return min(8 * NT, a.group - hc % a.chunks * (8 * NT));
  }
  // Output block md of accumulator fragments: rows are dims, columns 2c and 2c + 1 heads;
  // inv0 / inv1 normalise the two columns.
  __device__ static void store(const PagedArgs& a, int b, int hc, int nt, int md,
                               const float4& o, float inv0, float inv1, int lane) {
    const int g = lane >> 2, c = lane & 3, n = heads(a, hc);
    __nv_bfloat16* base = a.out + b * a.o_sb + static_cast<int64_t>(head0(a, hc)) * a.o_sh;
    if constexpr (kE4m3) {  // rows g and g + 8 are dims 2g and 2g + 1
      const int h = nt * 8 + 2 * c;
      // infinite only by a NaN in V: NaN again
      auto norm = [](float x, float inv) { return fmaf(x, 0.f, x * inv); };
      if (h < n)
        *reinterpret_cast<uint32_t*>(base + h * a.o_sh + md * 16 + 2 * g) =
            pack_bf16(norm(o.x, inv0), norm(o.z, inv0));
      if (h + 1 < n)
        *reinterpret_cast<uint32_t*>(base + (h + 1) * a.o_sh + md * 16 + 2 * g) =
            pack_bf16(norm(o.y, inv1), norm(o.w, inv1));
    } else {
      const uint32_t lo = transpose8x8(pack_bf16(o.x * inv0, o.y * inv1));
      const uint32_t hi = transpose8x8(pack_bf16(o.z * inv0, o.w * inv1));
      const int h = nt * 8 + g;
      if (h < n) {
        *reinterpret_cast<uint32_t*>(base + h * a.o_sh + md * 16 + 2 * c) = lo;
        *reinterpret_cast<uint32_t*>(base + h * a.o_sh + md * 16 + 8 + 2 * c) = hi;
      }
    }
  }
  __device__ static float inverse(const PagedArgs& a, int hc, float l) {
    const float unit = kE4m3 ? (a.v_scale ? a.v_scale[hc / a.chunks] : 1.f) / kWide : 1.f;
    return l == 0.f ? 0.f : unit / l;
  }
  __device__ static void store_lse(const PagedArgs& a, int b, int hc, int nt, float m0, float l0,
                                   float m1, float l1, int lane) {
    if (!a.lse || lane >= 4) return;
    const int h = nt * 8 + 2 * lane, n = heads(a, hc);
    float* base = a.lse + static_cast<int64_t>(b) * a.hq + head0(a, hc);
    constexpr float kLn2 = 0.693147180559945309f, shift = kE4m3 ? kF16Shift : 0.f;
    if (h < n) base[h] = l0 == 0.f ? -INFINITY : (m0 - shift) * kLn2 + logf(l0);
    if (h + 1 < n) base[h + 1] = l1 == 0.f ? -INFINITY : (m1 - shift) * kLn2 + logf(l1);
  }
};

// weight of a partial result with maximum m among ones with maximum `top`
__device__ __forceinline__ float weight_of(float m, float top) {
  return m == -INFINITY ? 0.f : exp2_fast(m - top);
}

// Sums of the threads before this one, and of the block; two barriers' worth of one.
template <int kWarps>
__device__ __forceinline__ int block_sums(int mine, int* s_warp_sum, int* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) s_warp_sum[warp] = upto;
  __syncthreads();
  int all = 0;
  upto -= mine;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) upto += all;
    all += s_warp_sum[w];
  }
  *total = all;
  return upto;
}

template <int D, bool kE4m3, int NT>
__global__ void __launch_bounds__(Shape<D, kE4m3, NT>::kWarps * 32, 1)
    paged_attn_kernel(PagedArgs a) {
  using S = Shape<D, kE4m3, NT>;
  using R = Rows<D, kE4m3, NT>;
  constexpr int kWarps = S::kWarps, kStages = S::kStages, kBlocks = S::kBlocks;
  constexpr int kThreads = kWarps * 32, MT = S::MT, kTile = S::kTile;
  // unsigned: rows may reach up to 2^31 - 16 tokens
  auto tiles_of = [](int len) {
    return static_cast<int>((static_cast<uint32_t>(len) + kTile - 1) / kTile);
  };
  extern __shared__ char smem[];
  char* const ring_mem = smem + (-smem_addr(smem) & 511u);  // rows lie on their own size
  // request (-1: no more tiles), segment, valid rows (a byte per subtile) and flags, tiles
  // left of the segment
  __shared__ int4 s_info[kWarps][kStages];
  constexpr int kRunLast = 1 << 16;
  __shared__ int4 s_begin[kWarps];          // request, segment, tile and request length at a
                                            // warp's start
  __shared__ int s_warp_sum[kWarps];
  __shared__ int4 s_tail[kWarps];  // has a tail | 2 starts it | 4 ends it, request, segment
  __shared__ Split s_split[kWarps];

  allow_dependent_launch();
  if (threadIdx.x < kWarps) s_begin[threadIdx.x] = make_int4(0, 0, 0, 0);
  wait_prerequisite();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hcs = a.hkv * a.chunks;  // segments per request

  const int first_worker = static_cast<int>(blockIdx.x) * kWarps;
  // ---- the line of tiles, and where each warp's run begins on it
  const int per = (a.batch + kThreads - 1) / kThreads;
  const int b0 = min(a.batch, static_cast<int>(threadIdx.x) * per), b1 = min(a.batch, b0 + per);
  int mine = 0, first_len = 0;
  for (int b = b0; b < b1; ++b) {
    const int n = a.lens[b];
    if (blockIdx.x == 0 && (n < 0 || n > a.max_len)) atomicOr(a.err, UMIC_DEVERR_BAD_PAGE);
    const int len = max(0, min(n, a.max_len));
    if (b == b0) first_len = len;
    mine += tiles_of(len);
  }
  int total;
  const int upto = block_sums<kWarps>(mine, s_warp_sum, &total);
  total *= hcs;
  const int workers = min(static_cast<int>(gridDim.x) * kWarps, total);
  const Line line(total, max(workers, 1));
  if (mine > 0 && first_worker < workers && line.begin(first_worker + kWarps) > upto * hcs) {
    for (int w = 0; w < kWarps && first_worker + w < workers; ++w) {
      int at = line.begin(first_worker + w) - upto * hcs;
      if (at < 0 || at >= mine * hcs) continue;
      for (int b = b0; b < b1; ++b) {
        const int len = b == b0 ? first_len : clamped_len(a, b), tiles = tiles_of(len);
        if (at < tiles * hcs) {
          s_begin[w] = make_int4(b, at / tiles, at % tiles, len);
          break;
        }
        at -= tiles * hcs;
      }
    }
  }
  // requests without tokens, dealt to the CTAs: zeros
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    if (clamped_len(a, b) > 0) continue;
    for (int i = threadIdx.x; i < a.hq * (D / 8); i += kThreads)
      st_vec(a.out + b * a.o_sb + i / (D / 8) * a.o_sh + i % (D / 8) * 8, make_uint4(0, 0, 0, 0));
    if (a.lse)
      for (int h = threadIdx.x; h < a.hq; h += kThreads)
        a.lse[static_cast<int64_t>(b) * a.hq + h] = -INFINITY;
  }
  __syncthreads();

  const int worker = first_worker + warp;
  int left = worker < workers ? line.begin(worker + 1) - line.begin(worker) : 0;  // to copy

  char* const ring = ring_mem + static_cast<size_t>(warp) * kStages * S::kTileBytes;
  const uint32_t ring_addr = smem_addr(ring);

  // ---- loader: the next tile to copy. Pages are looked up one tile ahead of their copies.
  int lb = 0, lhc = 0, lt = 0, ltiles = 0, lpi = 0, loff = 0, llen = 0;
  int page_id[MT], page_off[MT];
  // A lane holds one of 32 consecutive table entries, and the next 32, the row's first 32
  // (for the next head) and the next request's first 32 and length are under way: under
  // full load a dependent look-up takes microseconds.
  int entries = 0, entries_next = 0, entries_first = 0, other_entries = 0, other_len = 0;
  auto entry = [&](int b, int i) {
    return b < a.batch && i < a.max_pages ? a.table[b * a.table_stride + i] : 0;
  };
  auto fetch_other = [&]() {
    other_entries = entry(lb + 1, lane);
    other_len = lb + 1 < a.batch ? clamped_len(a, lb + 1) : 0;
  };
  auto look_up = [&]() {  // pages of tile lt; steps (lpi, loff) behind it
#pragma unroll
    for (int u = 0; u < MT; ++u) {
      page_off[u] = loff;
      page_id[u] = __shfl_sync(0xffffffffu, entries, lpi & 31);
      if ((loff += kSub) == a.page_size) {
        loff = 0;
        if ((++lpi & 31) == 0) {
          entries = entries_next;
          entries_next = entry(lb, lpi + 32 + lane);
        }
      }
    }
  };
  auto touch_q = [&]() {  // a new segment's q into L1, while its first tiles come
    const int n = R::heads(a, lhc);
    const char* q = reinterpret_cast<const char*>(
        a.q + lb * a.q_sb + static_cast<int64_t>(R::head0(a, lhc)) * a.q_sh);
    constexpr int kLines = (2 * D + 127) / 128;
    for (int i = lane; i < n * kLines; i += 32)
      asm volatile("prefetch.global.L1 [%0];" ::"l"(q + i / kLines * a.q_sh * 2 + i % kLines * 128));
  };
  const int4 start = left > 0 ? s_begin[warp] : make_int4(0, 0, 0, 0);
  if (left > 0) {
    lb = start.x;
    lhc = start.y;
    lt = start.z;
    llen = start.w;
    ltiles = tiles_of(llen);
    lpi = lt * kTile / a.page_size;
    loff = lt * kTile - lpi * a.page_size;
    entries = entry(lb, (lpi & ~31) + lane);
    entries_next = entry(lb, (lpi & ~31) + 32 + lane);
    entries_first = entry(lb, lane);
    fetch_other();
    look_up();
  }
  constexpr int kCols = S::kRow / 16;  // 16-byte pieces of a row
  constexpr int kCopies = (kSub * kCols + 31) / 32;
  const bool dense = a.pg_ss == S::kRow;  // a page's rows of a head lie one behind the other
  constexpr bool kEven = 32 % kCols == 0;  // 32 lanes copy whole rows
  const uint32_t lane_dst = S::piece(lane / kCols, lane % kCols);
  const int64_t v_minus_k = a.v_pages - a.k_pages;
  auto load = [&](int stage) {
    if (left > 0) {
      int rows_of = 0;
      const int64_t head_at = lhc / a.chunks * a.pg_sh;
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        int rows = max(0, min(kSub, llen - lt * kTile - u * kSub));
        int64_t page = page_id[u];
        if (page < 0 || page >= a.num_pages) {
          if (lane == 0 && rows > 0) atomicOr(a.err, UMIC_DEVERR_BAD_PAGE);
          page = 0;
          rows = 0;
        }
        rows_of |= rows << (8 * u);
        const char* k = a.k_pages + page * a.pg_sp + head_at + page_off[u] * a.pg_ss;
        const uint32_t dst = ring_addr + stage * S::kTileBytes + u * S::kSubBytes;
        if (kEven && dense && rows == kSub) {  // immediate offsets from two pointers
          const uint32_t to = dst + lane_dst;
          const char* at_k = k + lane * 16;
          const char* at_v = at_k + v_minus_k;
#pragma unroll
          for (int i = 0; i < kCopies; ++i) {
            const int row = i * (32 / kCols);  // of lane 0
            const uint32_t into = (S::kSwizzle ? to ^ ((row & 7) * 16) : to) + row * S::kPitch;
            cp_async16(into, at_k + i * 512);
            cp_async16(into + kSub * S::kPitch, at_v + i * 512);
          }
        } else {
          // rows behind the length are filled with zeros: a weight of 0 times what an
          // unwritten page holds could be NaN
#pragma unroll
          for (int i = 0; i < kCopies; ++i) {
            const int x = i * 32 + lane, row = x / kCols;
            const uint32_t to = dst + S::piece(row, x % kCols);
            if ((kSub * kCols) % 32 != 0 && x >= kSub * kCols) break;
            const char* at = k + row * a.pg_ss + x % kCols * 16;
            cp_async16(to, at, row < rows);
            cp_async16(to + kSub * S::kPitch, at + v_minus_k, row < rows);
          }
        }
      }
      --left;
      if (lane == 0) {
        s_info[warp][stage] = make_int4(lb, lhc, rows_of | (left == 0 ? kRunLast : 0), ltiles - lt);
      }
      if (left > 0) {
        if (++lt == ltiles) {
          lt = lpi = loff = 0;
          if (++lhc == hcs) {
            lhc = 0;
            ++lb;
            llen = other_len;
            entries_first = other_entries;
            if (llen == 0) {  // the requests behind an empty one are looked up in turn
              while (llen == 0 && lb + 1 < a.batch) llen = clamped_len(a, ++lb);
              entries_first = entry(lb, lane);
            }
            ltiles = tiles_of(llen);
            fetch_other();
          }
          entries = entries_first;
          entries_next = entry(lb, 32 + lane);
          touch_q();
        }
        look_up();
      }
    } else if (lane == 0) {
      s_info[warp][stage].x = -1;
    }
    cp_commit();
  };

  // ---- one segment's state
  const int g = lane >> 2, c = lane & 3;
  uint32_t qf[NT][kBlocks][2];
  float o[NT][kBlocks][4];
  float m[NT][2], l[NT][2], fac[NT][2];
  int sb = 0, shc = 0;

  auto begin_segment = [&](int b, int hc) {
    sb = b;
    shc = hc;
    const int n = R::heads(a, hc);
    const __nv_bfloat16* q = a.q + b * a.q_sb + static_cast<int64_t>(R::head0(a, hc)) * a.q_sh;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = nt * 8 + g;
      const __nv_bfloat16* row = q + h * a.q_sh;
      if constexpr (!kE4m3) {
#pragma unroll
        for (int k = 0; k < kBlocks; ++k) {
          qf[nt][k][0] = h < n ? *reinterpret_cast<const uint32_t*>(row + k * 16 + 2 * c) : 0u;
          qf[nt][k][1] = h < n ? *reinterpret_cast<const uint32_t*>(row + k * 16 + 8 + 2 * c) : 0u;
        }
        fac[nt][0] = fac[nt][1] = a.scale_log2;
      } else {
        // a lane's four bytes of a K row are dims 4c .. 4c + 3 of a block, widened as 4c,
        // 4c + 2 and 4c + 1, 4c + 3: q to match, as fp16, scaled by the power of two of the row's largest
        uint2 raw[kBlocks];
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < kBlocks; ++k) {
          raw[k] = h < n ? *reinterpret_cast<const uint2*>(row + k * 16 + 4 * c) : make_uint2(0, 0);
          top = fmaxf(top, fmaxf(fabsf(__uint_as_float(raw[k].x << 16)),
                                 fabsf(__uint_as_float(raw[k].x & 0xffff0000u))));
          top = fmaxf(top, fmaxf(fabsf(__uint_as_float(raw[k].y << 16)),
                                 fabsf(__uint_as_float(raw[k].y & 0xffff0000u))));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^e <= top < 2^(e + 1); e kept where 2^e and 2^-e are normal numbers
        const int e = max(-126, min(126, static_cast<int>(__float_as_uint(top) >> 23) - 127));
        const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        // an infinity in q makes every score of its head infinite or NaN, and the row NaN
        const float up = top < INFINITY ? __uint_as_float(static_cast<uint32_t>(127 + e) << 23)
                                        : NAN;
#pragma unroll
        for (int k = 0; k < kBlocks; ++k) {
          qf[nt][k][0] = pack_f16(__uint_as_float(raw[k].x << 16) * down,
                                  __uint_as_float(raw[k].y << 16) * down);
          qf[nt][k][1] = pack_f16(__uint_as_float(raw[k].x & 0xffff0000u) * down,
                                  __uint_as_float(raw[k].y & 0xffff0000u) * down);
        }
        const float f = a.scale_log2 * (a.k_scale ? a.k_scale[hc / a.chunks] : 1.f) / kWide * up;
        fac[nt][0] = __shfl_sync(0xffffffffu, f, 8 * c);
        fac[nt][1] = __shfl_sync(0xffffffffu, f, 8 * c + 4);
      }
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) o[nt][k][0] = o[nt][k][1] = o[nt][k][2] = o[nt][k][3] = 0.f;
    }
  };

  auto tile = [&](int stage, int rows_of) {
    const uint32_t at0 = ring_addr + stage * S::kTileBytes;
    // S^T in four accumulators, 4 / MT a subtile, to keep the chains of dependent products
    // short
    float s[NT][4][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[nt][x][j] = 0.f;
    const uint32_t k_at = at0 + S::piece((lane & 7) + (lane & 8), lane >> 4);
    if constexpr (!kE4m3) {
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) {
        uint32_t r[MT][4];
#pragma unroll
        for (int u = 0; u < MT; ++u) ldsm4(r[u], S::along(k_at + u * S::kSubBytes, k * 32));
#pragma unroll
        for (int u = 0; u < MT; ++u)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma_bf16(s[nt][MT == 2 ? 2 * u + (k & 1) : k & 3], r[u], qf[nt][k][0], qf[nt][k][1]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kBlocks; k += 2) {
#pragma unroll
        for (int u = 0; u < MT; ++u) {
          uint32_t r[4];
          const uint32_t at = S::along(k_at + u * S::kSubBytes, k * 16);
          if (k + 1 < kBlocks) ldsm4(r, at);
          else ldsm2(r[0], r[1], at);
#pragma unroll
          for (int x = 0; x < 2 && k + x < kBlocks; ++x) {
            uint32_t a0, a1, a2, a3;
            widen4(r[2 * x], a0, a2);
            widen4(r[2 * x + 1], a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma_f16(s[nt][MT == 2 ? 2 * u + x : (k + x) & 3], a0, a1, a2, a3, qf[nt][k + x][0],
                      qf[nt][k + x][1]);
          }
        }
      }
    }
    uint32_t ph[NT][MT][2], pl[NT][MT][2];  // P transposed: bf16 and its remainder, or fp16
    bool moved = false;
    float keep[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[MT][4], top[2] = {m[nt][0], m[nt][1]};
#pragma unroll
      for (int u = 0; u < MT; ++u) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float sum = MT == 2 ? s[nt][2 * u][j] + s[nt][2 * u + 1][j]
                                    : (s[nt][0][j] + s[nt][1][j]) + (s[nt][2][j] + s[nt][3][j]);
          x[u][j] = sum * fac[nt][j & 1];
          // infinite only by a NaN in K (widen4): a NaN score, not a weight of 0
          if constexpr (kE4m3) x[u][j] = fmaf(sum, 0.f, x[u][j]);
        }
        const int rows = rows_of >> (8 * u) & 255;
        if (rows < kSub) {
          if (g >= rows) x[u][0] = x[u][1] = -INFINITY;
          if (g + 8 >= rows) x[u][2] = x[u][3] = -INFINITY;
        }
        top[0] = fmaxf(top[0], fmaxf(x[u][0], x[u][2]));
        top[1] = fmaxf(top[1], fmaxf(x[u][1], x[u][3]));
      }
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], d));
        top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], d));
      }
      float ref[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        ref[j] = top[j] == -INFINITY ? 0.f : top[j];
        keep[nt][j] = exp2_fast(m[nt][j] - ref[j]);
        moved |= keep[nt][j] != 1.f;
        m[nt][j] = top[j];
        l[nt][j] *= keep[nt][j];
        if constexpr (kE4m3) ref[j] -= kF16Shift;
      }
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        float p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = exp2_fast(x[u][j] - ref[j & 1]);
        l[nt][0] += p[0] + p[2];
        l[nt][1] += p[1] + p[3];
        if constexpr (kE4m3) {
          ph[nt][u][0] = transpose8x8(pack_f16(p[0], p[1]));
          ph[nt][u][1] = transpose8x8(pack_f16(p[2], p[3]));
        } else {
          const uint32_t h0 = pack_bf16(p[0], p[1]), h1 = pack_bf16(p[2], p[3]);
          ph[nt][u][0] = transpose8x8(h0);
          ph[nt][u][1] = transpose8x8(h1);
          pl[nt][u][0] = transpose8x8(pack_bf16(p[0] - __uint_as_float(h0 << 16),
                                                p[1] - __uint_as_float(h0 & 0xffff0000u)));
          pl[nt][u][1] = transpose8x8(pack_bf16(p[2] - __uint_as_float(h1 << 16),
                                                p[3] - __uint_as_float(h1 & 0xffff0000u)));
        }
      }
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < kBlocks; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[nt][k][j] *= keep[nt][j & 1];
    }
    const uint32_t vt = at0 + kSub * S::kPitch;
    if constexpr (!kE4m3) {
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        const uint32_t at = vt + u * S::kSubBytes +
                            S::piece((lane & 7) + ((lane >> 4) << 3), (lane >> 3) & 1);
#pragma unroll
        for (int k0 = 0; k0 < kBlocks; k0 += 4) {
          uint32_t r[4][4];
#pragma unroll
          for (int k = 0; k < 4 && k0 + k < kBlocks; ++k) ldsm4t(r[k], S::along(at, (k0 + k) * 32));
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int k = 0; k < 4 && k0 + k < kBlocks; ++k)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const uint32_t (&p)[2] = y == 0 ? ph[nt][u] : pl[nt][u];
                mma_bf16(o[nt][k0 + k], r[k], p[0], p[1]);
              }
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        const uint32_t at =
            vt + u * S::kSubBytes + S::piece((lane & 7) + (lane & 8), lane >> 4);
#pragma unroll
        for (int k = 0; k < kBlocks; k += 2) {
          uint32_t r[4];
          if (k + 1 < kBlocks) ldsm4t(r, S::along(at, k * 16));
          else ldsm2t(r[0], r[1], S::along(at, k * 16));
#pragma unroll
          for (int x = 0; x < 2 && k + x < kBlocks; ++x) {
            // bytes: token 2c dims 2g, 2g + 1, token 2c + 1 the same
            uint32_t a0, a1, a2, a3;
            widen4(r[2 * x], a0, a1);
            widen4(r[2 * x + 1], a2, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma_f16(o[nt][k + x], a0, a1, a2, a3, ph[nt][u][0], ph[nt][u][1]);
          }
        }
      }
    }
  };

  auto sum_l = [&]() {  // the lanes' shares of the sums of weights
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], d);
  };
  auto store_slot = [&](float* dst) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < kBlocks; ++k)
        reinterpret_cast<float4*>(dst)[(nt * kBlocks + k) * 32 + lane] =
            make_float4(o[nt][k][0], o[nt][k][1], o[nt][k][2], o[nt][k][3]);
      if (lane < 4) {
        dst[S::kOut + nt * 8 + 2 * lane] = m[nt][0];
        dst[S::kOut + nt * 8 + 2 * lane + 1] = m[nt][1];
        dst[S::kOut + NT * 8 + nt * 8 + 2 * lane] = l[nt][0];
        dst[S::kOut + NT * 8 + nt * 8 + 2 * lane + 1] = l[nt][1];
      }
    }
  };

  // ---- the run
  int tail = 0;  // 1: a partial segment is left in registers, 2: it has the first tile, 4: the last
  Split split{-1, 0, 0, 0};
  if (worker < workers) {
#pragma unroll
    for (int i = 0; i < kStages; ++i) load(i);
    // the first segment's q comes while the first tiles do
    bool open = true, from_start = start.z == 0;
    begin_segment(start.x, start.y);
    int stage = 0, pos = line.begin(worker);  // place on the line
    while (true) {
      cp_wait<kStages - 1>();
      __syncwarp();
      const int4 info = s_info[warp][stage];
      if (info.x < 0) break;
      if (!open) {
        open = from_start = true;
        begin_segment(info.x, info.y);
      }
      ++pos;
      if (info.z & 0xffff) tile(stage, info.z);
      __syncwarp();
      load(stage);  // at once: no stage is empty while the warp waits for the next
      stage = stage + 1 == kStages ? 0 : stage + 1;
      const bool done = info.w == 1, run_ends = info.z & kRunLast;
      if (done || run_ends) {
        sum_l();
        open = false;
        if (done && from_start) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float i0 = R::inverse(a, shc, l[nt][0]), i1 = R::inverse(a, shc, l[nt][1]);
#pragma unroll
            for (int k = 0; k < kBlocks; ++k)
              R::store(a, sb, shc, nt, k,
                       make_float4(o[nt][k][0], o[nt][k][1], o[nt][k][2], o[nt][k][3]), i0, i1,
                       lane);
            R::store_lse(a, sb, shc, nt, m[nt][0], l[nt][0], m[nt][1], l[nt][1], lane);
          }
        } else if (!run_ends) {
          store_slot(a.ws.slot(worker, 1, S::kSlot));
        } else {
          tail = 1 | (from_start ? 2 : 0) | (done ? 4 : 0);
          if (from_start) {
            const int seg_end = pos + info.w - 1, last = line.run_of(seg_end - 1);
            split = Split{sb, shc, last, line.begin(last + 1) > seg_end};
          }
        }
      }
    }
    cp_wait<0>();
    __syncwarp();
    if (tail) store_slot(reinterpret_cast<float*>(ring));
  }
  if (lane == 0) {
    s_tail[warp] = make_int4(tail, sb, shc, 0);
    s_split[warp] = split;
  }
  __syncthreads();

  // ---- join the tails of this CTA: a run of warps from one that is not continued from its
  // left neighbour to the last one that continues it
  const int flags = lane < kWarps ? s_tail[lane].x : 0;
  const unsigned has = __ballot_sync(0xffffffffu, flags & 1);
  const unsigned first_tile = __ballot_sync(0xffffffffu, flags & 2);
  const unsigned last_tile = __ballot_sync(0xffffffffu, flags & 4);
  for (unsigned heads = has & (first_tile | 1u); heads; heads &= heads - 1) {
    const int w0 = __ffs(heads) - 1;
    const int w1 = w0 + __ffs(~((has & ~first_tile) >> (w0 + 1))) - 1;
    const int4 head = s_tail[w0];
    const bool whole = (first_tile >> w0 & 1) && (last_tile >> w1 & 1);
    float* const slot = a.ws.slot(first_worker + w0, 0, S::kSlot);
    for (int at = warp; at < NT * kBlocks; at += kWarps) {
      const int nt = at / kBlocks, k = at % kBlocks;
      float2 ms[kWarps], ls[kWarps];
      float4 vs[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {  // warps outside the run weigh nothing
        const float* p = reinterpret_cast<const float*>(
            ring_mem + static_cast<size_t>(min(max(w, w0), w1)) * kStages * S::kTileBytes);
        ms[w] = *reinterpret_cast<const float2*>(p + S::kOut + nt * 8 + 2 * c);
        ls[w] = *reinterpret_cast<const float2*>(p + S::kOut + NT * 8 + nt * 8 + 2 * c);
        vs[w] = reinterpret_cast<const float4*>(p)[at * 32 + lane];
      }
      float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        top[0] = fmaxf(top[0], ms[w].x);
        top[1] = fmaxf(top[1], ms[w].y);
      }
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w < w0 || w > w1) continue;
        const float x0 = weight_of(ms[w].x, top[0]), x1 = weight_of(ms[w].y, top[1]);
        sum[0] += x0 * ls[w].x;
        sum[1] += x1 * ls[w].y;
        acc.x += x0 * vs[w].x;
        acc.y += x1 * vs[w].y;
        acc.z += x0 * vs[w].z;
        acc.w += x1 * vs[w].w;
      }
      if (whole) {
        R::store(a, head.y, head.z, nt, k, acc, R::inverse(a, head.z, sum[0]),
                 R::inverse(a, head.z, sum[1]), lane);
        if (k == 0) R::store_lse(a, head.y, head.z, nt, top[0], sum[0], top[1], sum[1], lane);
      } else {
        reinterpret_cast<float4*>(slot)[at * 32 + lane] = acc;
        if (k == 0 && lane < 4) {
          slot[S::kOut + nt * 8 + 2 * lane] = top[0];
          slot[S::kOut + nt * 8 + 2 * lane + 1] = top[1];
          slot[S::kOut + NT * 8 + nt * 8 + 2 * lane] = sum[0];
          slot[S::kOut + NT * 8 + nt * 8 + 2 * lane + 1] = sum[1];
        }
      }
    }
    if (whole && threadIdx.x == 0) s_split[w0].b = -1;
  }
  __syncthreads();
  if (threadIdx.x < kWarps) a.ws.splits()[first_worker + threadIdx.x] = s_split[threadIdx.x];
}

// Running sum of partial results: (top, sum, acc) of two heads per lane.
struct Joined {
  float top0 = -INFINITY, top1 = -INFINITY, sum0 = 0.f, sum1 = 0.f;
  float4 acc = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(float m0, float m1, float l0, float l1, const float4& v) {
    const float t0 = fmaxf(top0, m0), t1 = fmaxf(top1, m1);
    const float a0 = weight_of(top0, t0), a1 = weight_of(top1, t1);
    const float b0 = weight_of(m0, t0), b1 = weight_of(m1, t1);
    sum0 = sum0 * a0 + l0 * b0;
    sum1 = sum1 * a1 + l1 * b1;
    acc.x = acc.x * a0 + v.x * b0;
    acc.y = acc.y * a1 + v.y * b1;
    acc.z = acc.z * a0 + v.z * b0;
    acc.w = acc.w * a1 + v.w * b1;
    top0 = t0;
    top1 = t1;
  }
};

constexpr int kJoinWarps = 4, kJoinBatch = 4, kJoinY = 8;

// Joins the partial results of the segments that cross runs. The splits left by the warps
// of the main kernel's CTA x belong to CTAs (x, 0 .. gridDim.y - 1). A split between two neighbours has two parts: one warp of
// those CTAs each, loading four output blocks of both at once. A longer one (up to every
// run, for one long request) is shared by the CTAs, output blocks y, y + gridDim.y, ...;
// its parts are dealt to the four warps, each loading four at a time, and joined in shared
// memory: the joining of 19 parts waits for memory twice, not 19 times.
template <int D, bool kE4m3, int NT>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(PagedArgs a) {
  using S = Shape<D, kE4m3, NT>;
  using R = Rows<D, kE4m3, NT>;
  constexpr int kWarps = S::kWarps, kAll = NT * S::kBlocks;
  __shared__ float4 s_acc[kJoinWarps][32];
  __shared__ float4 s_ml[kJoinWarps][32];
  allow_dependent_launch();
  wait_prerequisite();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & 3;
  const int first = blockIdx.x * kWarps;
  int4 mine = make_int4(-1, 0, 0, 0);
  if (lane < kWarps) mine = reinterpret_cast<const int4*>(a.ws.splits())[first + lane];
  // parts between the first run's and the last one's: one of every further CTA
  const int mid_mine = (mine.z - mine.w) / kWarps - static_cast<int>(blockIdx.x);
  const unsigned near = __ballot_sync(0xffffffffu, mine.x >= 0 && mid_mine == 0);
  unsigned far = __ballot_sync(0xffffffffu, mine.x >= 0 && mid_mine > 0);

  auto top_of = [&](const float* p, int nt) {
    return *reinterpret_cast<const float2*>(p + S::kOut + nt * 8 + 2 * c);
  };
  auto sum_of = [&](const float* p, int nt) {
    return *reinterpret_cast<const float2*>(p + S::kOut + NT * 8 + nt * 8 + 2 * c);
  };
  auto finish = [&](const Joined& j, int b, int hc, int nt, int k) {
    R::store(a, b, hc, nt, k, j.acc, R::inverse(a, hc, j.sum0), R::inverse(a, hc, j.sum1), lane);
    if (k == 0) R::store_lse(a, b, hc, nt, j.top0, j.sum0, j.top1, j.sum1, lane);
  };

  unsigned left = near;
  for (int turn = 0; left; ++turn, left &= left - 1) {
    const int i = __ffs(left) - 1;
    const int b = __shfl_sync(0xffffffffu, mine.x, i), hc = __shfl_sync(0xffffffffu, mine.y, i);
    const int last = __shfl_sync(0xffffffffu, mine.z, i);
    if (turn % (kJoinWarps * kJoinY) != static_cast<int>(blockIdx.y) * kJoinWarps + warp) continue;
    const float *p = a.ws.slot(first + i, 0, S::kSlot), *q = a.ws.slot(last, 1, S::kSlot);
#pragma unroll 1
    for (int nt = 0; nt < NT; ++nt) {
      const float2 pm = top_of(p, nt), pl = sum_of(p, nt), qm = top_of(q, nt), ql = sum_of(q, nt);
#pragma unroll 1
      for (int k0 = 0; k0 < S::kBlocks; k0 += kJoinBatch) {
        float4 x[kJoinBatch], y[kJoinBatch];
#pragma unroll
        for (int u = 0; u < kJoinBatch; ++u) {
          const int at = (nt * S::kBlocks + min(k0 + u, S::kBlocks - 1)) * 32 + lane;
          x[u] = reinterpret_cast<const float4*>(p)[at];
          y[u] = reinterpret_cast<const float4*>(q)[at];
        }
#pragma unroll
        for (int u = 0; u < kJoinBatch; ++u) {
          if (k0 + u >= S::kBlocks) break;
          Joined j;
          j.add(pm.x, pm.y, pl.x, pl.y, x[u]);
          j.add(qm.x, qm.y, ql.x, ql.y, y[u]);
          finish(j, b, hc, nt, k0 + u);
        }
      }
    }
  }
  for (; far; far &= far - 1) {
    const int i = __ffs(far) - 1;
    const int b = __shfl_sync(0xffffffffu, mine.x, i), hc = __shfl_sync(0xffffffffu, mine.y, i);
    const int last = __shfl_sync(0xffffffffu, mine.z, i);
    const int head = __shfl_sync(0xffffffffu, mine.w, i);
    const int mid = __shfl_sync(0xffffffffu, mid_mine, i);
    const int parts = 1 + mid + head;
    auto part = [&](int x) -> const float* {  // in line order
      const int run = x == 0 ? first + i
                      : x > mid ? last : (static_cast<int>(blockIdx.x) + x) * kWarps;
      return a.ws.slot(run, x > mid ? 1 : 0, S::kSlot);
    };
#pragma unroll 1
    for (int at = blockIdx.y; at < kAll; at += gridDim.y) {
      const int nt = at / S::kBlocks;
      Joined j;
#pragma unroll 1
      for (int x0 = warp; x0 < parts; x0 += kJoinWarps * kJoinBatch) {
        float2 m[kJoinBatch], l[kJoinBatch];
        float4 v[kJoinBatch];
#pragma unroll
        for (int u = 0; u < kJoinBatch; ++u) {  // all loads first; absent parts are left out
          const float* p = part(min(x0 + u * kJoinWarps, parts - 1));
          m[u] = top_of(p, nt);
          l[u] = sum_of(p, nt);
          v[u] = reinterpret_cast<const float4*>(p)[at * 32 + lane];
        }
#pragma unroll
        for (int u = 0; u < kJoinBatch; ++u)
          if (x0 + u * kJoinWarps < parts) j.add(m[u].x, m[u].y, l[u].x, l[u].y, v[u]);
      }
      s_acc[warp][lane] = j.acc;
      s_ml[warp][lane] = make_float4(j.top0, j.top1, j.sum0, j.sum1);
      __syncthreads();
      if (warp == 0) {
        Joined all;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w)
          all.add(s_ml[w][lane].x, s_ml[w][lane].y, s_ml[w][lane].z, s_ml[w][lane].w,
                  s_acc[w][lane]);
        finish(all, b, hc, nt, at % S::kBlocks);
      }
      __syncthreads();
    }
  }
}

// Query heads that share a segment: 8, or 16 for wider groups, which halves the K and V
// traffic of their segments (256 requests of up to 4096 tokens, 16 query heads to each of 4 KV
// heads x 128: 200 us against 325 with 8, e4m3 167 against 205; head_dim 256 keeps 8:
// accumulators of 16 would not fit the registers, and 16 query heads to a KV head take 329 us,
// 0.48 of measured HBM).
int heads_per_segment(int group, int head_dim) { return group > 8 && head_dim <= 128 ? 16 : 8; }

// CTAs of the main kernel: one per SM, fewer where the longest line that the table allows is
// shorter.
int64_t ctas_of(int64_t batch, int hkv, int group, int head_dim, bool e4m3, int64_t max_len) {
  const int tile = subtiles(head_dim, e4m3) * kSub, per = heads_per_segment(group, head_dim);
  const int warps = warps_per_cta(head_dim, e4m3, per);
  const int64_t tiles = (max_len + tile - 1) / tile * batch * hkv * ((group + per - 1) / per);
  return std::max<int64_t>(1, std::min<int64_t>(sm_count(), (tiles + warps - 1) / warps));
}

template <int D, bool kE4m3, int NT>
void launch(PagedArgs a, cudaStream_t st) {
  using S = Shape<D, kE4m3, NT>;
  a.chunks = (a.group + 8 * NT - 1) / (8 * NT);
  const unsigned ctas =
      static_cast<unsigned>(ctas_of(a.batch, a.hkv, a.group, D, kE4m3, a.max_len));
  a.ws.runs = static_cast<int64_t>(ctas) * S::kWarps;
  static std::once_flag once[64];
  int dev = 0;
  cudaGetDevice(&dev);
  std::call_once(once[dev & 63], [] {
    cudaFuncSetAttribute(paged_attn_kernel<D, kE4m3, NT>,
                         cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kSmem));
  });
  prefer_max_shared<paged_join_kernel<D, kE4m3, NT>>();
  launch_pdl(paged_attn_kernel<D, kE4m3, NT>, dim3(ctas), dim3(S::kWarps * 32), S::kSmem, st, a);
  launch_pdl(paged_join_kernel<D, kE4m3, NT>, dim3(ctas, kJoinY), dim3(kJoinWarps * 32), 0, st, a);
}

template <int D>
void launch_d(const PagedArgs& a, bool e4m3, cudaStream_t st) {
  if constexpr (D <= 128) {
    if (heads_per_segment(a.group, D) == 16) {
      if (e4m3) launch<D, true, 2>(a, st);
      else launch<D, false, 2>(a, st);
      return;
    }
  }
  if (e4m3) launch<D, true, 1>(a, st);
  else launch<D, false, 1>(a, st);
}

}  // namespace
}  // namespace umic

using namespace umic;

extern "C" size_t umic_paged_attention_workspace_bytes(int64_t batch, int32_t hq, int32_t hkv,
                                                       int32_t head_dim, int64_t max_pages,
                                                       int64_t page_size, int cache_dtype) {
  if (batch <= 0 || hq <= 0 || hkv <= 0 || head_dim <= 0 || max_pages < 0 || page_size <= 0 ||
      hq / hkv == 0)
    return 0;
  const bool e4m3 = cache_dtype == UMIC_DTYPE_E4M3;
  const int per = heads_per_segment(hq / hkv, head_dim);
  return Space::bytes(ctas_of(batch, hkv, hq / hkv, head_dim, e4m3, max_pages * page_size) *
                          warps_per_cta(head_dim, e4m3, per),
                      per * (head_dim + 2));
}

extern "C" int umic_paged_attention(const umic_paged_attention_args* args, void* stream) {
  const char* const me = "umic_paged_attention";
  clear_error();
  if (!args) return fail(UMIC_ERR_INVALID_ARG, "%s: null pointer", me);
  const auto& [q, k_pages, v_pages, k_scale, v_scale, block_table, kv_lens, out, lse,
               workspace, q_sb, q_sh, pg_sp, pg_sh, pg_ss, num_pages, page_size,
               table_stride, max_pages, o_sb, o_sh, batch, workspace_bytes, hq, hkv,
               head_dim, cache_dtype, scale] = *args;
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
  // tiles of every segment, had every request the longest row, count in 32 bits
  const int64_t segments = static_cast<int64_t>(batch) * hkv * ((hq / hkv + 7) / 8);
  if (segments > 0x3fffffffLL / std::max<int64_t>(1, max_pages * page_size / kSub))
    return fail(UMIC_ERR_UNSUPPORTED,
                "%s: batch * KV heads * max_pages * page_size / 16 must stay below 2^30", me);
  if (batch == 0) return UMIC_OK;
  if (!q || !k_pages || !v_pages || !kv_lens || !out || (max_pages > 0 && !block_table))
    return fail(UMIC_ERR_INVALID_ARG, "%s: null pointer", me);
  const int64_t pe = cache_dtype == UMIC_DTYPE_E4M3 ? 16 : 8;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out) ||
      q_sb % 8 || q_sh % 8 || o_sb % 8 || o_sh % 8 || pg_sp % pe || pg_sh % pe || pg_ss % pe)
    return fail(UMIC_ERR_ALIGNMENT, "%s: 16-byte alignment of bases / strides", me);
  if (!rows_apart({{batch, o_sb}, {hq, o_sh}}, head_dim))
    return fail(UMIC_ERR_INVALID_ARG, "%s: output rows overlap", me);
  const size_t need = umic_paged_attention_workspace_bytes(batch, hq, hkv, head_dim, max_pages,
                                                           page_size, cache_dtype);
  if (!workspace || !aligned16(workspace) || workspace_bytes < static_cast<int64_t>(need))
    return fail(UMIC_ERR_INVALID_ARG, "%s: workspace of %lld bytes (%zu needed, 16-byte aligned)",
                me, (long long)workspace_bytes, need);
  uint32_t* err = device_error_word();
  if (!err) return fail(UMIC_ERR_DEVICE, "%s: no device error word", me);
  const bool e4m3 = cache_dtype == UMIC_DTYPE_E4M3;
  const int64_t es = e4m3 ? 1 : 2;
  PagedArgs a{};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.k_pages = static_cast<const char*>(k_pages);
  a.v_pages = static_cast<const char*>(v_pages);
  a.k_scale = e4m3 ? k_scale : nullptr;
  a.v_scale = e4m3 ? v_scale : nullptr;
  a.table = block_table;
  a.lens = kv_lens;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.lse = lse;
  a.err = err;
  a.ws.base = static_cast<char*>(workspace);
  a.q_sb = q_sb; a.q_sh = q_sh; a.o_sb = o_sb; a.o_sh = o_sh;
  a.pg_sp = pg_sp * es; a.pg_sh = pg_sh * es; a.pg_ss = pg_ss * es;
  a.table_stride = table_stride;
  a.max_len = static_cast<int32_t>(max_pages * page_size);
  a.max_pages = static_cast<int32_t>(max_pages);
  a.num_pages = num_pages;
  a.page_size = static_cast<int32_t>(page_size);
  a.hq = hq; a.hkv = hkv; a.batch = static_cast<int32_t>(batch); a.group = hq / hkv;
  a.scale_log2 = scale * 1.4426950408889634f;
  cudaStream_t st = as_stream(stream);
  if (head_dim == 64) launch_d<64>(a, e4m3, st);
  else if (head_dim == 80) launch_d<80>(a, e4m3, st);
  else if (head_dim == 96) launch_d<96>(a, e4m3, st);
  else if (head_dim == 128) launch_d<128>(a, e4m3, st);
  else launch_d<256>(a, e4m3, st);
  return launch_status(me);
}
