// Attention over a paged cache where a request may have more rows than the narrow kernel takes: prompts, chunks of them, drafts of many
// heads, and whatever else is in such a batch (single tokens among chunks: their memory time passes under the chunks' arithmetic).
//
// Rows are (new token, query head) pairs of one KV head, a token's heads next to one another, so that a K or V tile serves all heads of
// the group.  A CTA takes up to 256 rows over tiles of 128 positions, with two accumulators of 128 rows:
//
//   warp 8       streams K and V tiles, page by page, by TMA (128-byte swizzle, no multicast) into a ring of four
//   warps 9, 10  issue tcgen05.mma, w = 0 and 1: S_w = Q K^T into tensor memory, and O_w += P_w V with P_w from tensor memory.  One warp
//                for both spent as long on waits, fences and commits between the products as the tensor cores on these
//   warps 0-3, 4-7   softmax w = 0, 1, one row a thread: S out of tensor memory, maximum, weights, sum, P back over S
//   warp 11      walks the span, hands out its items and brings their rows of Q
//
// Items of more than 128 rows: accumulator w is rows 128 w .. of the item, over the same tiles of positions.  Items of up to 128: both have
// the same rows, accumulator w the w-th half of every tile, and are added at the end.
//
// Scores come by halves of a tile, 64 positions, into two sets of columns in turn: while a softmax is at one half, the products of the
// half before and the scores of the one behind run, so that neither waits for the way there and back (arrival, wait, issue and commit are
// 350 clocks by themselves; with one buffer of 128 positions the chain of scores, softmax and outputs took 5300 clocks a pair of
// tiles).  Tensor memory is full: 2 x 2 x 64 columns S (P over its first half, 16 bits), 2 x 128 columns O.  S(i + 2) is issued behind O(i) by the
// same thread, so "S is there" says that P(i) has been read and O(i) added.
//
// The running maximum is only moved when it grows by more than 2^8: till then weights are up to 256 instead of 1, which fp32 sums and
// 16-bit weights hold alike (relative rounding), and O is left alone.
//
// Where rows are many no one unit bounds it.  A pair of accumulators over a tile is 2048 clocks of tensor cores, 2560 of shared memory (192 KB
// read for the scores, Q again for every 64 positions, 64 for the outputs, 64 written by TMA, at 128 bytes each) and 1536 of exponentials (2048, a
// quarter of them by polynomial), and about 4100 pass.  Prompts, 396 us when it was measured: 371 without the softmax's arithmetic, 359 with an
// eighth of the products, 249 with neither; so the greater part is the way between the two, arrivals, waits, loads and stores of tensor
// memory and issue, twice a tile as scores come by halves.  One buffer of 128 positions an accumulator whose weights are handed over in
// parts has not been tried.  Where rows are few, it is bound by memory and the way from one item to the next.  Prompts of up to 4096 tokens, 397 GFLOP:
// 393 us, 1010 TFLOP/s (435 - 475 us under the power cap); a chunk of 512 tokens at 16384, 34.9 GFLOP: 47.6 us, 8 of them the join of
// pieces; 24 requests of 5 tokens, 103 MB: 32 us; a chunk of 2047 tokens among 23 single ones, 107 GFLOP and 234 MB: 146 us.
#pragma once

#include "paged_work.cuh"

namespace b200ipc {

constexpr int kWideRows = 256;
constexpr int kWideTile = 128;   // positions
constexpr int kWideHalf = 64;
constexpr int kWideStages = 4;   // K or V tiles
constexpr int kWideThreads = 384;  // three warpgroups
constexpr int kWideTileBytes = kWideTile * kAttnD * 2;  // also of 128 rows of Q
constexpr int kWideStage = 4096;  // bytes of a softmax warp's way out: 32 rows x 128
constexpr size_t kWideSmem = 1024 + size_t(kWideStages + 2) * kWideTileBytes + 8 * kWideStage;
// What an item's start and end cost, in positions.  A chunk of 512 tokens at 16384: 55.0 us with 96, 52.8 with 192, 50.7 with 384, no less with more.
constexpr int kWideStart = 384;
constexpr int kWideLeast = 576;  // a span is at least so long: more than kWideStart + a tile, so that every cut leaves a tile on both sides
constexpr float kWideSlack = 8.f;
// Every so manieth pair of weights is computed on the other units: prompts of up to 4096 tokens 416 us without, 395 with every fourth, 436 with
// every second.
constexpr int kWidePoly = 4;

// The part of an item that lies in a span.
struct WideItem {
  int valid;
  int request, h;       // KV head
  int first, n, len;    // the request's first row of q, its new tokens, its tokens in the cache
  int row0, rows;       // rows of the item within the request
  int t0, t1, whole;    // tiles of positions; whether these are all
  int split;            // up to 128 rows: the accumulators take a half of every tile each
  int count[2];         // halves of tiles that accumulator w looks at
};

struct WideCut {
  const PagedArgs& a;
  __device__ __forceinline__ bool takes(const Request& r) const { return r.n > 0; }
  __device__ __forceinline__ int items(const Request& r) const { return (r.n * a.group + kWideRows - 1) / kWideRows; }
  // positions that the rows below `rows` of the request see
  __device__ __forceinline__ int seen(const Request& r, int rows) const {
    return rows <= 0 ? 0 : max(0, r.len - r.n + (min(rows, r.n * a.group) - 1) / a.group + 1);
  }
  __device__ __forceinline__ int tiles(const Request& r, int item) const { return (seen(r, (item + 1) * kWideRows) + kWideTile - 1) / kWideTile; }
  // Length of the first `t` items of a head, in positions x group: item u sees max(len - n, 0) + (u + 1) * 256 / group positions or a few less.
  __device__ __forceinline__ uint64_t before(const Request& r, uint32_t t) const {
    return uint64_t(t) * (uint32_t(max(0, r.len - r.n) + kWideStart) * uint64_t(a.group) + (kWideRows / 2) * (t + 1));
  }
  __device__ __forceinline__ uint64_t length(const Request& r) const { return takes(r) ? uint32_t(a.hkv) * before(r, uint32_t(items(r))) : 0; }
  __device__ __forceinline__ Start start(const Request& r, int request, int h, int item, int n, int tile) const {
    return Start{request, h * n + item, tile, h, item * kWideRows, min(kWideRows, r.n * a.group - item * kWideRows), r};
  }
  __device__ __forceinline__ Start place(const Request& r, int request, uint64_t offset) const {
    const int n = items(r);
    const uint64_t per = before(r, uint32_t(n));
    int h = 0;
    while (offset >= per) {  // a few heads
      offset -= per;
      ++h;
    }
    int lo = 0, hi = n;  // the last item that begins at or before it
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before(r, uint32_t(mid)) <= offset) lo = mid;
      else hi = mid;
    }
    const uint64_t in = offset - before(r, uint32_t(lo)), skip = uint64_t(kWideStart) * uint32_t(a.group);
    const int t = in <= skip ? 0 : int(divide(in - skip + uint64_t(kWideTile / 2) * uint32_t(a.group), uint32_t(kWideTile * a.group)));
    const int all = tiles(r, lo);
    if (t >= all && all > 0) {  // rounded to its end: the next item
      if (lo + 1 < n) return start(r, request, h, lo + 1, n, 0);
      if (h + 1 < a.hkv) return start(r, request, h + 1, 0, n, 0);
      return Start{request + 1};
    }
    return start(r, request, h, lo, n, min(t, max(all - 1, 0)));
  }
};

// The span's items one after the other.
struct WideWalk {
  const PagedArgs& a;
  const WideCut cut;
  const Start last;
  Window win;
  int i, number, t0;
  __device__ __forceinline__ WideWalk(const PagedArgs& args, const Start& first, const Start& end)
      : a(args), cut{args}, last(end), i(first.request), number(first.number), t0(first.tile) {}
  __device__ __forceinline__ WideItem next() {
    WideItem x{};
    const auto takes = [&](const Request& r) { return cut.takes(r); };
    if (i < a.requests) {
      const int found = win.next(a, i, takes);
      if (found != i) {  // a mark may stand on a request that is not this kernel's, behind one that is
        i = found;
        number = t0 = 0;
      }
    }
    if (i >= a.requests || i > last.request || (i == last.request && (number > last.number || (number == last.number && t0 >= last.tile)))) return x;
    x.valid = 1;
    const Request r = win.get(i);
    const int n = cut.items(r);
    x.request = i;
    x.h = number / n;
    x.first = r.row0;
    x.n = r.n;
    x.len = r.len;
    const int item = number - x.h * n;
    x.row0 = item * kWideRows;
    x.rows = min(kWideRows, r.n * a.group - x.row0);
    const int tiles = cut.tiles(r, item);
    x.t0 = t0;
    x.t1 = i == last.request && number == last.number ? last.tile : tiles;
    x.whole = t0 == 0 && x.t1 == tiles;
    x.split = x.rows <= 128;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      if (x.split) {
        x.count[w] = x.t1 - x.t0;
      } else {
        const int see = cut.seen(r, x.row0 + min(x.rows, (w + 1) * 128));
        x.count[w] = 2 * max(0, min((see + kWideTile - 1) / kWideTile, x.t1) - x.t0);
      }
    }
    t0 = 0;
    if (++number == a.hkv * n) {
      number = 0;
      ++i;
    }
    return x;
  }
};

__device__ __forceinline__ void tmem_st_16cols(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// The left operand (128 rows, 16 columns of 16 bits) from tensor memory
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Right operand whose columns (dimensions) lie next to one another: blocks of 64 columns, 128-byte rows in the 128-byte swizzle, a
// kWideTileBytes / 2 apart; groups of eight rows (positions) 1024 bytes apart.
__device__ __forceinline__ uint64_t make_sw128_nmajor_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= uint64_t((smem_addr & 0x3ffffu) >> 4);
  d |= uint64_t((kWideTileBytes / 2) >> 4) << 16;
  d |= uint64_t(1024 >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(2) << 61;
  return d;
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 64 columns x `group` heads x 128 / group tokens of Q: 128 rows of the item
__device__ __forceinline__ void tma_load_5d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int half, int h, int token) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(half), "r"(0), "r"(h), "r"(token)
      : "memory");
}
// Two fp32 values in one register pair
__device__ __forceinline__ uint64_t f32x2(float a, float b) {
  uint64_t x;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a), "f"(b));
  return x;
}
__device__ __forceinline__ float2 f32x2_parts(uint64_t x) {
  float2 y;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(y.x), "=f"(y.y) : "l"(x));
  return y;
}
__device__ __forceinline__ uint64_t f32x2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t x;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(x) : "l"(a), "l"(b), "l"(c));
  return x;
}
__device__ __forceinline__ uint64_t f32x2_add(uint64_t a, uint64_t b) {
  uint64_t x;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(x) : "l"(a), "l"(b));
  return x;
}
// NaN where one of them is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float m;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
// 2^x for two values up to 127, without the special function unit: x = n + f with |f| <= 1/2, 2^f by the polynomial 1 + f q(f) of degree 4 whose
// greatest relative error there is least (3.6e-6, found by Remez' exchange), n into the exponent.  From -127 down, -inf included, it is zero (the bits
// of 1 less 127 in the exponent), between -127 and -126 what is below 2^-126; what NaN gives is no number to go by.
__device__ __forceinline__ float2 exp2_poly(uint64_t x) {
  float2 v = f32x2_parts(x);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(v.x) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(v.y) : "f"(-127.f));
  x = f32x2(v.x, v.y);
  constexpr float kWhole = 12582912.f;  // 3 x 2^22: behind the addition the last bits are n
  const uint64_t t = f32x2_add(x, f32x2(kWhole, kWhole));
  const uint64_t f = f32x2_fma(f32x2_add(t, f32x2(-kWhole, -kWhole)), f32x2(-1.f, -1.f), x);
  uint64_t p = f32x2_fma(f, f32x2(0.009782912209630013f, 0.009782912209630013f), f32x2(0.055976882576942444f, 0.055976882576942444f));
  p = f32x2_fma(p, f, f32x2(0.24020710587501526f, 0.24020710587501526f));
  p = f32x2_fma(p, f, f32x2(0.6931136250495911f, 0.6931136250495911f));
  p = f32x2_fma(p, f, f32x2(1.f, 1.f));
  const float2 y = f32x2_parts(p), n = f32x2_parts(t);
  return make_float2(__int_as_float(__float_as_int(y.x) + (__float_as_int(n.x) << 23)), __int_as_float(__float_as_int(y.y) + (__float_as_int(n.y) << 23)));
}

__device__ __forceinline__ void cp_async_16(uint32_t smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(gmem) : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kWideThreads, 1) paged_wide_kernel(const __grid_constant__ PagedArgs args) {
  extern __shared__ unsigned char smem_raw[];
  using Items = Queue<WideItem, 11>;  // the softmax warps, the stream, the products
  __shared__ Items s_queue;
  __shared__ uint64_t kv_full[kWideStages], kv_empty[kWideStages], q_ready[2], q_free[2], s_full[2][2], p_ready[2][2], o_late[2], o_full[2], mma_done;
  __shared__ float2 s_ml[128];  // maxima and sums of w = 1
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ uint64_t s_sum[kWideThreads / 32];
  __shared__ Start s_span[2];
  __shared__ Axis s_axis;
  unsigned char* q_smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* ring = q_smem + 2 * kWideTileBytes;
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = int(threadIdx.x & 31);
  volatile int* abort_flag = &s_abort;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kWideStages; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 2);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&q_ready[w], 1);
      mbar_init(&q_free[w], 2);
      mbar_init(&s_full[w][0], 1);
      mbar_init(&s_full[w][1], 1);
      mbar_init(&o_late[w], 1);
      mbar_init(&p_ready[w][0], 4);  // a warp is one arrival: 128 on one word would stand in line
      mbar_init(&p_ready[w][1], 4);
      mbar_init(&o_full[w], 1);
    }
    mbar_init(&mma_done, 2);
    s_queue.init();
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }
  __syncwarp();
  tc_fence_before_sync();
  pdl_wait();
  const WideCut cut{args};
  find_span<kWideThreads>(
      args, [&](const Request& r) { return cut.length(r); }, [&](const Request& r, int i, uint64_t o) { return cut.place(r, i, o); },
      uint32_t(kWideLeast * args.group), s_sum, s_span, &s_axis);
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = s_tmem;
  QueueEnd<Items, WideItem> items{s_queue, abort_flag, args.timeout_ns};
  auto wait = [&](uint64_t* bar, uint32_t parity) { items.wait(bar, parity); };
  auto wait_warp = [&](uint64_t* bar, uint32_t parity) { items.wait_warp(bar, parity); };

  if (warp < 8) {
    // ---- softmax: thread = row of the accumulator -----------------------------------------------------------------------
    const int w = warp >> 2, row = (warp & 3) * 32 + lane, G = args.group;
    const uint32_t lane_base = tmem + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t s_addr = lane_base + uint32_t(w) * 128u, o_addr = lane_base + 256u + uint32_t(w) * 128u;
    uint32_t part_no = 0, ph_o = 0, ring_at = 0;  // halves of tiles so far, and the ring's tiles before the item
    for (const WideItem* x = items.take(); x != nullptr; x = items.take()) {
      // What is needed once is read or computed again: the loop over the tiles has few registers to spare.
      const int count = x->count[w], G0 = x->split ? 0 : w * 128;  // first row of this accumulator in the item
      float ref = -INFINITY, sum = 0;  // the maximum that the weights are taken against (log2 domain)
      if (G0 < x->rows) {
        const bool busy = G0 + (warp & 3) * 32 < x->rows;  // this warp has rows
        // positions that this row sees
        const int limit = G0 + row < x->rows ? x->len - x->n + (x->row0 + G0 + row) / G + 1 : 0;
        const int step = x->split ? kWideTile : kWideHalf;
        int p0 = x->t0 * kWideTile + (x->split ? w * kWideHalf : 0);
        for (int i = 0; i < count; ++i, p0 += step) {
          const uint32_t b = part_no & 1u;
          wait_warp(&s_full[w][b], (part_no >> 1) & 1u);
          ++part_no;
          // Values of positions that do not exist count as zero (a weight of zero would not do: they may be NaN).  They are in the item's last
          // tile; each softmax that uses it clears them, as neither waits for the other.
          if (p0 + kWideHalf > x->len) {
            const uint32_t v_at = ring_at + uint32_t(2 * (x->t1 - x->t0) - 1), v_st = v_at % kWideStages;  // that tile in the ring
            wait_warp(&kv_full[v_st], (v_at / kWideStages) & 1u);
            const int at = row & (kWideHalf - 1), first = p0 & (kWideTile - 1);  // two threads a position, half of its dimensions each
            if (p0 + at >= x->len) {
              unsigned char* v = ring + v_st * kWideTileBytes + (first + at) * 128 + (row >= kWideHalf ? kWideTileBytes / 2 : 0);
#pragma unroll
              for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(v + (c << 4)) = make_uint4(0, 0, 0, 0);
            }
            fence_async_smem();
          }
          if (busy) {
            tc_fence_after_sync();
            const uint32_t s_at = s_addr + b * kWideHalf;
            float s[kWideHalf];
#pragma unroll
            for (int c = 0; c < 2; ++c) tmem_ld_32cols(s_at + uint32_t(c) * 32u, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * c]));
            tmem_ld_wait();
            if (__any_sync(0xffffffffu, limit < p0 + kWideHalf)) {
#pragma unroll
              for (int e = 0; e < kWideHalf; ++e)
                if (p0 + e >= limit) s[e] = -INFINITY;
            }
            float mx[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = max3(s[e], s[e + 4], s[e + 8]);
#pragma unroll
            for (int e = 12; e < kWideHalf; e += 2) mx[(e >> 1) & 3] = max3(mx[(e >> 1) & 3], s[e], s[e + 1]);
            const float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]) * args.scale_log2;
            if (__any_sync(0xffffffffu, top > ref + kWideSlack)) {
              const float now = fmaxf(ref, top);
              if (i > 0) {
                // O(i - 1) has to be there: what says so is S(i + 1), or, for the last one, a word of its own
                if (i + 1 < count) wait_warp(&s_full[w][b ^ 1u], (part_no >> 1) & 1u);
                else wait_warp(&o_late[w], ph_o);
                tc_fence_after_sync();
                const float f = now == -INFINITY ? 1.f : exp2_fast(ref - now);
                sum *= f;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                  uint32_t o[16];
                  tmem_ld_16cols(o_addr + uint32_t(c) * 16u, o);
                  tmem_ld_wait();
#pragma unroll
                  for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                  tmem_st_16cols(o_addr + uint32_t(c) * 16u, o);
                }
              }
              ref = now;
            }
            const float shift = ref == -INFINITY ? 0.f : -ref;
            uint64_t part[2] = {0, 0};  // pairs of sums
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              uint32_t p[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const uint64_t v = f32x2_fma(f32x2(s[32 * c + 2 * e], s[32 * c + 2 * e + 1]), f32x2(args.scale_log2, args.scale_log2), f32x2(shift, shift));
                float2 y;
                if (e % kWidePoly == kWidePoly - 1) {
                  y = exp2_poly(v);
                } else {
                  y = f32x2_parts(v);
                  y = make_float2(exp2_fast(y.x), exp2_fast(y.y));
                }
                part[e & 1] = f32x2_add(part[e & 1], f32x2(y.x, y.y));
                p[e] = pack2<T>(y.x, y.y);
              }
              tmem_st_16cols(s_at + uint32_t(c) * 16u, p);
            }
            tmem_st_wait();
            tc_fence_before_sync();
            const float2 a = f32x2_parts(f32x2_add(part[0], part[1]));
            // A score of NaN or +inf (inf - inf) makes the row NaN.  The sum has to say so: exp2_poly does not.
            sum = top < INFINITY ? sum + (a.x + a.y) : __int_as_float(0x7fffffff);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_ready[w][b]);
        }
      }
      // ---- the end of the item ---------------------------------------------------------------------------------------------------
      const bool split = x->split != 0, whole = x->whole != 0, both = split && x->t1 > x->t0;
      const bool busy = G0 + (warp & 3) * 32 < x->rows, exists = G0 + row < x->rows;
      const int at = x->row0 + G0 + row, j = at / G;
      if (count > 0) {
        wait_warp(&o_full[w], ph_o);
        ph_o ^= 1u;
        tc_fence_after_sync();
      }
      // Rows leave by 128 bytes: through 4 KB of the warp's own, 16-byte chunks swapped by row, eight lanes a row.  (A row a lane, as the
      // accumulator comes, is 32 lines for every store, and cost 8 us an item.)
      unsigned char* way = ring + kWideStages * kWideTileBytes + warp * kWideStage;
      char* const mine = whole ? reinterpret_cast<char*>(static_cast<T*>(args.out) + (int64_t(x->first + j) * args.hq + int64_t(x->h) * G + (at - j * G)) * kAttnD)
                               : reinterpret_cast<char*>(Piece<kWideRows>::slot(args, int(blockIdx.x), x->t0 > 0 ? 0 : 1) + 2 * kWideRows + size_t(G0 + row) * kAttnD);
      const int first_row = G0 + (warp & 3) * 32, rows = x->rows;
      auto leave = [&](int bytes) {  // what is in the warp's memory goes to `bytes` behind each row's start
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = i * 4 + (lane >> 3);
          char* to = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), r));
          const uint4 v = *reinterpret_cast<const uint4*>(way + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
          if (first_row + r < rows) *reinterpret_cast<uint4*>(to + bytes + (lane & 7) * 16) = v;
        }
        __syncwarp();
      };
      auto chunk = [&](int c) { return reinterpret_cast<uint4*>(way + lane * 128 + ((c ^ (lane & 7)) << 4)); };
      auto put = [&](const uint32_t (&o)[32], int c) {  // dimensions c .. c + 31
        if (whole) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            auto two = [&](int k) { return pack2<T>(__uint_as_float(o[e + 2 * k]), __uint_as_float(o[e + 2 * k + 1])); };
            *chunk(((c & 32) + e) >> 3) = make_uint4(two(0), two(1), two(2), two(3));
          }
          if (c & 32) leave((c & 64) * 2);
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 4) *chunk(e >> 2) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          leave(c * 4);
        }
      };
      // Where both accumulators have the same rows, w = 0 adds them: every warp can read its 32 rows of all of tensor memory.
      float f = 1, g = 0;
      if (both) {
        if (w == 1) {
          s_ml[row] = make_float2(ref, sum);
          tc_fence_before_sync();
        }
        meet<256>();
        tc_fence_after_sync();
        const float2 other = s_ml[row];
        const float m = fmaxf(ref, other.x), u = m == -INFINITY ? 0.f : m;
        f = exp2_fast(ref - u);
        g = exp2_fast(other.x - u);
        sum = sum * f + other.y * g;
        ref = m;
      }
      if ((!split || w == 0) && busy) {
        if (exists && !whole) *reinterpret_cast<float2*>(Piece<kWideRows>::slot(args, int(blockIdx.x), x->t0 > 0 ? 0 : 1) + 2 * (G0 + row)) = make_float2(sum == 0 && x->len - x->n + j >= 0 ? kNoWeight : ref, sum);
        float none = 0;  // for a row without a weight
        if (whole) {
          if (sum == 0) none = no_weight(x->len - x->n + j >= 0);
          const float inv = sum == 0 ? 0.f : 1 / sum;
          f *= inv;
          g *= inv;
        }
#pragma unroll 1
        for (int c = 0; c < kAttnD; c += 32) {
          uint32_t o[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(none);
          if (count > 0) {
            tmem_ld_32cols(o_addr + uint32_t(c), o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(f != 0 && sum != 0 ? __uint_as_float(o[e]) * f : none);
          }
          if (both) {
            uint32_t y[32];
            tmem_ld_32cols(o_addr + 128u + uint32_t(c), y);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) + (g != 0 && sum != 0 ? __uint_as_float(y[e]) * g : 0.f));
          }
          put(o, c);
        }
      }
      tc_fence_before_sync();  // O may be written again once this thread's next weights are there
      if (both) meet<256>();   // of w = 1 as well
      ring_at += uint32_t(2 * (x->t1 - x->t0));
      items.give_back();
    }
    while (!meet<256>(true)) {
    }
  } else {
    if (warp == 8) {
      // ---- the stream: K and V of a tile after the other.  Lane l knows where box l of it is. -------------------------------
      const int box_log = min(args.page_log, 6), box = 1 << box_log, boxes_log = 7 - box_log, boxes = 1 << boxes_log, per_page = args.page_log - box_log;
      uint32_t st = 0, ph = 0;
      int issued = 0;
      auto load = [&](const CUtensorMap* map, int at, int n) {
        wait_warp(&kv_empty[st], ph ^ 1u);
        if (__any_sync(0xffffffffu, *abort_flag)) return;
        const int sent = args.mute && blockIdx.x == 0 && issued == 0 ? 0 : n;
        if (lane == 0 && sent > 0) mbar_expect_tx(&kv_full[st], uint32_t(n << box_log) * kAttnD * 2u);
        __syncwarp();
        unsigned char* dst = ring + st * kWideTileBytes;
        for (int k = 0; k < sent; ++k, dst += box * 128) {
          const int row = __shfl_sync(0xffffffffu, at, k);
          if (elect_one()) {
            tma_load_2d(dst, map, &kv_full[st], 0, row);
            tma_load_2d(dst + kWideTileBytes / 2, map, &kv_full[st], 64, row);
          }
          __syncwarp();
        }
        ++issued;
        if (++st == kWideStages) {
          st = 0;
          ph ^= 1u;
        }
      };
      for (const WideItem* x = items.take(); x != nullptr; x = items.take()) {
        const int* table = args.table + int64_t(x->request) * args.width;
        const int len = x->len, h = x->h, t1 = x->t1, pages = (len + (1 << args.page_log) - 1) >> args.page_log;
        int base = -64, entry = 0;  // 32 entries of the request's table, one per lane
        for (int t = x->t0; t < t1; ++t) {
          const int b0 = t << boxes_log;
          if (((b0 + boxes - 1) >> per_page) >= base + 32) {
            base = b0 >> per_page;
            entry = base + lane < pages ? table[base + lane] : -1;
          }
          const int at = box_row(args, h, b0 + (lane & (boxes - 1)), box_log, entry, base);
          const int n = min(boxes, (len - t * kWideTile + box - 1) >> box_log);  // boxes that hold positions of the request
          load(&args.tma_k, at, n);
          load(&args.tma_v, at, n);
        }
        items.give_back();
      }
      const uint64_t since = globaltimer_ns();
      for (int back = 1; back <= min(issued, kWideStages); ++back)
        mbar_drain(&kv_full[(issued - back) % kWideStages], uint32_t((issued - back) / kWideStages) & 1u, since);
    } else if (warp < 11) {
      // ---- the products of accumulator w: one thread ---------------------------------------------------------------------------
      if (elect_one()) {
        const int w = warp - 9;
        const uint32_t idesc_s = make_idesc<T>(128, kWideHalf), idesc_o = make_idesc<T>(128, kAttnD) | (1u << 16);
        const uint32_t t_s = tmem + uint32_t(w) * 128u, t_o = t_s + 256u;
        // 64 columns of a K-major tile are one block of it, 16 of them 32 bytes of its rows; descriptors count in 16 bytes
        const uint64_t q_desc = make_sw128_kmajor_desc(smem_u32(q_smem)), k_desc = make_sw128_kmajor_desc(smem_u32(ring)), v_desc = make_sw128_nmajor_desc(smem_u32(ring));
        constexpr uint64_t kTileStep = kWideTileBytes >> 4, kBlockStep = kWideTileBytes >> 5;
        uint32_t ph_q0 = 0, ph_q1 = 0;
        uint32_t base = 0, seen = 0;     // tiles of the ring before the item, and those that have landed
        uint32_t scored = 0, added = 0;  // halves of tiles whose S, whose O has been issued
        for (const WideItem* x = items.take_alone(); x != nullptr; x = items.take_alone()) {
          const uint32_t end = base + 2u * uint32_t(x->t1 - x->t0), last = added + uint32_t(x->count[w]), first = added;
          const bool split = x->split != 0;
          const uint32_t shift = split ? 0u : 1u;  // two halves of a tile, or one
          wait(&q_ready[0], ph_q0);
          ph_q0 ^= 1u;
          if (!split) {
            wait(&q_ready[1], ph_q1);
            ph_q1 ^= 1u;
            mbar_arrive(&q_free[1 - w]);  // the other's, seen
          }
          const uint64_t q = q_desc + uint64_t(split ? 0 : w) * kTileStep;
          uint64_t* q_done = &q_free[split ? 0 : w];
          if (first == last) mbar_arrive(q_done);
          // The ring has K and V of a tile after the other.  Scores are issued up to two halves ahead of the outputs, as soon as K is there; outputs
          // as soon as V and the weights are.  (One after the other in a fixed order, a wait for the next K held up what frees the ring for it.)
          // Both threads look for every tile in order, and both give it back, also where only one uses it: copies land out of order, and a wait
          // for a stage's next round must come from who has seen the round before, and find the round it looks for still there.
          uint64_t since = 0;
          uint32_t idle = 0;
          while (added < last || seen < end) {
            ++idle;
            if (seen < end && mbar_try_wait(&kv_full[seen % kWideStages], (seen / kWideStages) & 1u, 0)) {
              if (((seen - base) >> 1) >= ((last - first) >> shift)) mbar_arrive(&kv_empty[seen % kWideStages]);  // not this accumulator's
              ++seen;
              idle = 0;
            }
            if (scored < last && scored < added + 2) {
              const uint32_t tile = (scored - first) >> shift, k_at = base + 2 * tile;
              if (seen > k_at) {
                const uint32_t b = scored & 1u, half = split ? uint32_t(w) : (scored - first) & 1u;
                const uint64_t k = k_desc + uint64_t(k_at % kWideStages) * kTileStep + uint64_t(half) * (kWideHalf * 128 / 16);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const uint64_t o = uint64_t(i >> 2) * kBlockStep + uint64_t(i & 3) * 2u;
                  umma_f16(t_s + b * kWideHalf, q + o, k + o, idesc_s, i > 0 ? 1u : 0u);
                }
                umma_commit(&s_full[w][b]);
                if (split || half == 1) umma_commit(&kv_empty[k_at % kWideStages]);
                if (++scored == last) umma_commit(q_done);  // behind its last reader
                idle = 0;
              }
            }
            if (added < scored) {
              const uint32_t tile = (added - first) >> shift, v_at = base + 2 * tile + 1, b = added & 1u;
              if (seen > v_at && mbar_try_wait(&p_ready[w][b], (added >> 1) & 1u, 0)) {
                const uint32_t half = split ? uint32_t(w) : (added - first) & 1u;
                const uint64_t v = v_desc + uint64_t(v_at % kWideStages) * kTileStep + uint64_t(half) * (kWideHalf / 16 * 128);
                tc_fence_after_sync();
#pragma unroll
                for (int i = 0; i < kWideHalf / 16; ++i)  // 16 positions: 8 columns of P, 2048 bytes of V
                  umma_f16_ts(t_o, t_s + b * kWideHalf + uint32_t(i * 8), v + uint64_t(i) * 128u, idesc_o, added > first || i > 0 ? 1u : 0u);
                if (split || half == 1) umma_commit(&kv_empty[v_at % kWideStages]);
                ++added;
                if (added + 1 == last || last - first == 1) umma_commit(&o_late[w]);  // once an item
                if (added == last) umma_commit(&o_full[w]);
                idle = 0;
              }
            }
            if ((idle & 1023u) == 1023u) {  // nothing for a while
              const uint64_t now = globaltimer_ns();
              if (idle == 1023u) since = now;
              if (*abort_flag || now - since > args.timeout_ns) {
                *abort_flag = 1;
                break;
              }
            }
          }
          base = end;
          items.give_back_alone();
        }
        umma_commit(&mma_done);
        mbar_drain(&mma_done, 0, globaltimer_ns());
      }
      __syncwarp();
    } else {
      // ---- the walk, and Q: by TMA where a tile of 128 rows is whole tokens, else 16 lanes a row, one 16-byte chunk each -----------
      const Start first_item = s_span[0], last = s_span[1];
      if (lane == 0) {
        args.starts[blockIdx.x] = first_item;
        if (blockIdx.x == gridDim.x - 1) args.starts[gridDim.x] = last;
      }
      WideWalk walk(args, first_item, last);
      uint32_t ph[2] = {1, 1};
      int sent[2] = {0, 0};
      for (;;) {
        const WideItem x = walk.next();
        if (!items.put(x)) break;
        const int G = args.group;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (w * 128 >= x.rows) continue;
          wait_warp(&q_free[w], ph[w]);
          ph[w] ^= 1u;
          if (__any_sync(0xffffffffu, *abort_flag)) continue;
          if (args.q_boxes) {
            if (elect_one()) {
              mbar_expect_tx(&q_ready[w], kWideTileBytes);
              for (int half = 0; half < 2; ++half)
                tma_load_5d(q_smem + w * kWideTileBytes + half * (kWideTileBytes / 2), &args.tma_q, &q_ready[w], half, x.h, x.first + (x.row0 + w * 128) / G);
            }
            __syncwarp();
            ++sent[w];
          } else {
            const int c = lane & 15;
            const uint32_t to = smem_u32(q_smem) + uint32_t(w) * kWideTileBytes + uint32_t(c >> 3) * (kWideTileBytes / 2);
            const T* base = static_cast<const T*>(args.q) + int64_t(x.first) * args.row_stride + int64_t(x.h) * G * kAttnD + c * 8;
            for (int r = w * 128 + (lane >> 4); r < min(x.rows, (w + 1) * 128); r += 2) {
              const int j = (x.row0 + r) / G, in = r & 127;
              cp_async_16(to + uint32_t(in) * 128u + uint32_t(((c & 7) ^ (in & 7)) << 4), base + int64_t(j) * args.row_stride + (x.row0 + r - j * G) * kAttnD);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_ready[w]);
          }
        }
      }
      const uint64_t since = globaltimer_ns();
#pragma unroll
      for (int w = 0; w < 2; ++w)
        if (sent[w] > 0) mbar_drain(&q_ready[w], uint32_t(sent[w] - 1) & 1u, since);
    }
  }
  __syncwarp();
  zero_tail<T>(args);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 9) tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && *abort_flag) atomicOr(args.status, kPagedGaveUp);
}

}  // namespace b200ipc
