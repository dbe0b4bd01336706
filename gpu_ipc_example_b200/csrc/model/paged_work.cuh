// What the kernels of the attention over a paged cache share: their arguments, how the work is cut, and the kernel that joins the pieces.
//
// An item is what one CTA can do by itself: the query rows of a (request, KV head) (narrow kernel), or a tile of them (wide kernel), over
// the positions they see, in tiles of positions.  All items follow one another on one axis, each as long as its tiles and a constant for
// its start and end; the axis is cut into equal spans, one per CTA (one per SM).  So nobody waits for a longest request, and a single long
// one uses the whole GPU.  Every CTA finds its span itself from the lengths on the GPU: one round of loads and a scan, and the same
// rounding everywhere.  One warp of it then walks the span and hands the items to the others through a queue in shared memory.
//
// An item that a cut goes through leaves pieces: fp32 sums, maxima and unscaled outputs in the workspace.  A CTA has at most two, the end
// of an item that began in an earlier span (slot 0) and the beginning of one that goes on in the next (slot 1); they are joined in that
// order, so the result does not depend on timing: by the CTA that is done last where they are small (narrow kernel), by a kernel of its own
// where one SM would be at it for microseconds.
#pragma once

#include "../common/check.h"
#include "../fused/gemm_local.cuh"
#include "decode_math.cuh"
#include "paged_ops.h"

namespace b200ipc {

constexpr int kPagedQueue = 4;                    // items handed out ahead

struct Request {
  int row0, n, len;  // first row of q, new tokens, tokens in the cache
};

// Where a span starts: on tile `tile` of an item, and what the walking warp and the join have to know of that.
struct Start {
  int request, number, tile;  // number: of the request's items, KV head by KV head
  int h, row0, rows;          // of the item: KV head, first row within the request, rows
  Request r;
  uint64_t origin;            // where on the axis the item begins (narrow kernel)
};
// The axis: `spans` of `per`, the first `more` of them longer by one.
struct Axis {
  uint64_t per;
  uint32_t spans, more;
};

struct PagedArgs {
  alignas(64) CUtensorMap tma_k, tma_v;  // [pages * hkv * page, 128], boxes of 64 columns x min(page, 64) rows
  alignas(64) CUtensorMap tma_q;         // [rows, hkv, group, 2, 64], boxes of 128 (row, head) pairs x 64 columns; wide kernel only
  const void* q;
  void* out;
  const int *table, *lens, *cu_new;
  Start* starts;    // [CTAs + 1]; wide kernel
  unsigned int* arrived;  // [CTAs]: pieces of the item that begins in this span and goes on; zero between calls; narrow kernel
  float* part;      // [CTAs][2] pieces
  int* status;      // what went wrong since it was zeroed (bits)
  int64_t row_stride;
  int rows, requests, hq, hkv, group, max_new;
  int page_log, width;  // positions of a page: a power of two
  int64_t pages;
  int q_boxes;      // whether tma_q is there: 128 is a multiple of the group
  uint64_t timeout_ns;  // of one wait inside a CTA, which takes microseconds
  int mute;         // CTA 0's first copies into its ring are left out (failure injection)
  float scale_log2;
};

// 2^x in one instruction: relative error 2^-22, results below 2^-126 are zero.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ Request request_at(const PagedArgs& a, int i) {
  Request r;
  const int from = a.cu_new[i], to = a.cu_new[i + 1], len = a.lens[i];
  r.row0 = min(max(from, 0), a.rows);
  r.n = min(max(to, r.row0), a.rows) - r.row0;
  r.len = min(max(len, 0), a.width << a.page_log);
  return r;
}

// A warp's view of 32 requests, one per lane.
struct Window {
  int base = -64;
  Request mine;
  __device__ __forceinline__ void load(const PagedArgs& a, int i) {
    base = i;
    const int at = i + int(threadIdx.x & 31);
    mine = at < a.requests ? request_at(a, at) : Request{0, 0, 0};
  }
  // the first request from i on that `takes`, or a.requests
  template <typename Takes>
  __device__ __forceinline__ int next(const PagedArgs& a, int i, Takes takes) {
    while (i < a.requests) {
      if (i < base || i >= base + 32) load(a, i);
      const unsigned found = __ballot_sync(0xffffffffu, takes(mine)) & (0xffffffffu << (i - base));
      if (found) return base + __ffs(int(found)) - 1;
      i = base + 32;
    }
    return a.requests;
  }
  __device__ __forceinline__ Request get(int i) const {
    return {__shfl_sync(0xffffffffu, mine.row0, i - base), __shfl_sync(0xffffffffu, mine.n, i - base), __shfl_sync(0xffffffffu, mine.len, i - base)};
  }
};

// x / y, where x mostly fits 32 bits
__device__ __forceinline__ uint64_t divide(uint64_t x, uint32_t y) {
  return (x >> 32) == 0 ? uint64_t(uint32_t(x) / y) : x / y;
}
// Where this CTA's span starts and ends, into s_span.  All threads of the block; a barrier has to follow.  `length` of a request: its part of
// the axis, 0 for one that is not this kernel's; `place`: where on it an offset is.  No span is shorter than `least` but where the axis ends.
// Code that runs once runs at the speed at which it is fetched (20 clocks an instruction and more), so there is as little of it as
// can be, the same for all warps, and no division of 64 bits (300 clocks) unless the axis is that long.  s_sum: THREADS / 32 words.
template <int THREADS, typename Length, typename Place>
__device__ __forceinline__ void find_span(const PagedArgs& a, Length length, Place place, uint32_t least, uint64_t* s_sum, Start* s_span, Axis* s_axis) {
  const int lane = int(threadIdx.x & 31), warp = int(threadIdx.x >> 5);
  const int each = (a.requests + THREADS - 1) / THREADS;  // one, mostly
  const int i0 = min(a.requests, int(threadIdx.x) * each), i1 = min(a.requests, i0 + each);
  Request r{0, 0, 0};
  uint64_t mine = 0;
  for (int i = i0; i < i1; ++i) {
    r = request_at(a, i);
    mine += length(r);
    if (r.n > a.max_new && blockIdx.x == 0) atomicOr(a.status, kPagedMoreNew);
  }
  uint64_t in = mine;
#pragma unroll 1
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t x = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) in += x;
  }
  if (lane == 31) s_sum[warp] = in;
  if (threadIdx.x < 2) s_span[threadIdx.x] = Start{a.requests};
  __syncthreads();
  uint64_t before = in - mine, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
  }
  const uint32_t spans = uint32_t(min(uint64_t(gridDim.x), max(uint64_t(1), divide(total, least))));
  const uint64_t per = divide(total, spans);
  const uint32_t more = uint32_t(total - per * spans);
  if (threadIdx.x == 0) *s_axis = Axis{per, spans, more};
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const uint32_t c = blockIdx.x + uint32_t(k);
    const uint64_t at = c < spans ? per * c + min(c, more) : total;
    if (at >= before && at < before + mine) {
      uint64_t o = at - before;
      int i = i0;
      if (each > 1) {
        for (;; ++i) {
          r = request_at(a, i);
          const uint64_t l = length(r);
          if (o < l) break;
          o -= l;
        }
      }
      s_span[k] = place(r, i, o);
      s_span[k].origin += at - o;
    }
  }
}

// The span that a place on the axis is in.
__device__ __forceinline__ int span_of(const Axis& a, uint64_t x) {
  const uint64_t longer = (a.per + 1) * a.more;
  return x < longer ? int(divide(x, uint32_t(a.per + 1))) : int(a.more + divide(x - longer, uint32_t(a.per)));
}

// The queue: the walking warp fills a place, READERS warps give it back.
template <typename Item, int READERS>
struct Queue {
  uint64_t full[kPagedQueue], empty[kPagedQueue];
  Item items[kPagedQueue];
  __device__ void init() {
    for (int i = 0; i < kPagedQueue; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], READERS);
    }
  }
};
// The box of a cache's tensor map that is box `b` of a request's tiles (boxes of 1 << box_log positions), one lane each: `entry` holds 32
// entries of its table from `base` on.  A page that the cache does not have is a box outside of it.
__device__ __forceinline__ int box_row(const PagedArgs& a, int h, int b, int box_log, int entry, int base) {
  const int page = b >> (a.page_log - box_log);
  const int64_t id = __shfl_sync(0xffffffffu, entry, page - base);
  const int64_t at = id >= 0 && id < a.pages ? (id * a.hkv + h) << a.page_log : (a.pages * a.hkv) << a.page_log;
  return int(at) + (id >= 0 && id < a.pages ? (b << box_log) & ((1 << a.page_log) - 1) : 0);
}
// One warp's place in it.
template <typename Q, typename Item>
struct QueueEnd {
  Q& q;
  volatile int* abort_flag;
  uint64_t timeout_ns;
  uint32_t at = 0, ph = 0;
  __device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity) {
    if (!mbar_try_wait(bar, parity) && !*abort_flag) mbar_wait(bar, parity, abort_flag, timeout_ns);
  }
  // The same by all lanes of a warp, which leave it together: what follows may be instructions of the whole warp.
  __device__ __forceinline__ void wait_warp(uint64_t* bar, uint32_t parity) {
    wait(bar, parity);
    __syncwarp();
  }
  __device__ __forceinline__ void step() {
    if (++at == kPagedQueue) {
      at = 0;
      ph ^= 1u;
    }
  }
  // nullptr behind the last item
  __device__ __forceinline__ const Item* take() {
    wait_warp(&q.full[at], ph);
    const Item* x = &q.items[at];
    return x->valid && !__any_sync(0xffffffffu, *abort_flag) ? x : nullptr;
  }
  __device__ __forceinline__ void give_back() {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&q.empty[at]);
    step();
  }
  // The same for one thread by itself
  __device__ __forceinline__ const Item* take_alone() {
    wait(&q.full[at], ph);
    const Item* x = &q.items[at];
    return x->valid && !*abort_flag ? x : nullptr;
  }
  __device__ __forceinline__ void give_back_alone() {
    mbar_arrive(&q.empty[at]);
    step();
  }
  // false when nothing more is wanted.  Behind a wait that ran out the place may still be read, so it stays as it is: half of one item and half of
  // another would be rows that are not there.
  __device__ __forceinline__ bool put(const Item& x) {
    wait_warp(&q.empty[at], ph ^ 1u);
    if (__any_sync(0xffffffffu, *abort_flag)) return false;
    if ((threadIdx.x & 31) == 0) {
      q.items[at] = x;
      mbar_arrive(&q.full[at]);
    }
    __syncwarp();
    step();
    return x.valid != 0;
  }
};

// A barrier of the THREADS that compute; true once all of them are leaving.  After a wait that ran out some may leave an item before others, which
// would stand at a plain barrier for good: who leaves goes on meeting the others until they leave too.
template <int THREADS>
__device__ __forceinline__ bool meet(bool leaving = false) {
  uint32_t all;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.and.pred p, 1, %2, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(all)
               : "r"(uint32_t(leaving)), "n"(THREADS)
               : "memory");
  return all != 0;
}

// A piece: [rows] pairs (maximum in the log2 domain, sum), then [rows][128] of the output, not divided by the sum.  Where the sum is zero the wide
// kernel's maximum is kNoWeight for a row that sees positions, all of whose scores here are -inf, and -inf for a row that sees none: the join
// has that from the piece (from the lengths it would be a round to memory more, 2 us).
constexpr float kNoWeight = -3.4028234663852886e38f;
template <int ROWS>
struct Piece {
  static constexpr size_t kFloats = size_t(ROWS) * (2 + kAttnD);
  __device__ static float* slot(const PagedArgs& a, int cta, int which) { return a.part + (size_t(cta) * 2 + size_t(which)) * kFloats; }
};

// At the end of both kernels, all threads: rows behind the last request are zeros.
template <typename T>
__device__ __forceinline__ void zero_tail(const PagedArgs& a) {
  const int tail = min(max(a.cu_new[a.requests], 0), a.rows), vectors = a.hq * kAttnD / 8;
  for (int64_t row = int64_t(tail) + blockIdx.x; row < a.rows; row += gridDim.x)
    for (int v = int(threadIdx.x); v < vectors; v += int(blockDim.x))
      reinterpret_cast<uint4*>(static_cast<T*>(a.out) + row * a.hq * kAttnD)[v] = make_uint4(0, 0, 0, 0);
}

// What a row without a weight (a sum of zero) is: zero where it sees no position, 0 / 0 where it sees some and all their scores are -inf.
__device__ __forceinline__ float no_weight(bool sees) { return sees ? __int_as_float(0x7fffffff) : 0.f; }
__device__ __forceinline__ float4 divided(const float4& o, float l, bool sees) {
  if (l == 0) {
    const float x = no_weight(sees);
    return make_float4(x, x, x, x);
  }
  const float inv = 1 / l;
  return make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// ---- the join ---------------------------------------------------------------------------------------------------------
// Where an item starts in span c = blockIdx.x and goes on in the next, its pieces are weighted with 2^(maximum - greatest maximum) and added
// in order.  Eight rows a CTA, a warp each, whatever the pieces.  (All warps for one row after the other are as many rounds of loads behind one another,
// and barriers besides: one request of 5 tokens x 8 heads at 32000, in 148 pieces, 37 us a call so, 26 with a warp each.)  Registers for four
// pieces on their way at a time: with 32 a thread, which the compiler takes by itself, 28 us.
constexpr int kJoinThreads = 256;
constexpr int kJoinRows = kJoinThreads / 32;
struct Joined {
  float m = -INFINITY, l = 0;
  float4 o = make_float4(0, 0, 0, 0);
  __device__ __forceinline__ void add(const float2& ml, const float4& v) {
    const float now = fmaxf(m, ml.x), u = now == -INFINITY ? 0.f : now;
    const float c0 = exp2_fast(m - u), c1 = exp2_fast(ml.x - u);
    m = now;
    l = l * c0 + ml.y * c1;
    o = make_float4(o.x * c0 + v.x * c1, o.y * c0 + v.y * c1, o.z * c0 + v.z * c1, o.w * c0 + v.w * c1);
  }
};
template <typename T, int ROWS>
__global__ void __launch_bounds__(kJoinThreads, 6) paged_join_kernel(const __grid_constant__ PagedArgs a, int spans) {
  pdl_launch_dependents();
  pdl_wait();
  const int c = int(blockIdx.x), warp = int(threadIdx.x >> 5), lane = int(threadIdx.x & 31);
  const Start here = a.starts[c], next = a.starts[c + 1];
  int k = c + 2 + int(threadIdx.x);  // where the spans behind start
  Start from = k <= spans ? a.starts[k] : Start{-1};
  const int row0 = int(blockIdx.y) * kJoinRows;
  if (next.tile == 0 || (here.request == next.request && here.number == next.number && here.tile > 0) || row0 >= next.rows) return;
  int pieces = 2;  // one in this span, and in each of the following ones that start inside of the item
  for (int base = c + 2; base <= spans; base += kJoinThreads) {
    pieces += __syncthreads_count(from.request == next.request && from.number == next.number && from.tile > 0);
    k += kJoinThreads;
    from = k <= spans ? a.starts[k] : Start{-1};
  }
  const int row = row0 + warp;
  if (row >= next.rows) return;
  Joined x;
#pragma unroll 4
  for (int n = 0; n < pieces; ++n) {
    const float* p = Piece<ROWS>::slot(a, c + n, n == 0 ? 1 : 0);
    x.add(__ldcg(reinterpret_cast<const float2*>(p + 2 * row)), __ldcg(reinterpret_cast<const float4*>(p + 2 * ROWS + size_t(row) * kAttnD + lane * 4)));
  }
  const int at = next.row0 + row, j = at / a.group;
  const float4 y = divided(x.o, x.l, x.m > -INFINITY);
  T* dst = static_cast<T*>(a.out) + (int64_t(next.r.row0 + j) * a.hq + int64_t(next.h) * a.group + (at - j * a.group)) * kAttnD + lane * 4;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(y.x, y.y), pack2<T>(y.z, y.w));
}

}  // namespace b200ipc
