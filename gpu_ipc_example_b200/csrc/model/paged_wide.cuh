// Attention over a paged cache for requests with many rows: prompts, and chunks of them.
//
// Rows are (new token, query head) pairs of one KV head, a token's heads next to one another, so that a K or V tile serves all heads of
// the group.  A CTA takes 256 rows, two accumulator tiles of 128, over tiles of 128 positions:
//
//   warp 8       streams K and V tiles, page by page, by TMA (128-byte swizzle, no multicast) into a ring of five
//   warp 10      walks the span and hands its items to the others through a queue in shared memory
//   warp 9       issues tcgen05.mma: S_w = Q_w K^T into tensor memory, and O_w += P_w V with P_w from tensor memory
//   warps 0-3, 4-7   softmax of tile w = 0, 1, one row a thread: S out of tensor memory, maximum, weights, sum, P back over S
//
// While one tile's softmax runs, the tensor cores work for the other.  Tensor memory is full: 2 x 128 columns S (P over it, 16 bits), 2 x
// 128 columns O.  The running maximum is only moved when it grows by more than 2^8: till then weights are up to 256 instead of 1, which
// fp32 sums and 16-bit weights hold alike (relative rounding), and O is left alone (fetching and storing it costs as much as the softmax
// of a tile).  The order of S_w(j + 1) behind O_w(j) in the one issuing thread is what makes both "P has been read" and "O is complete"
// follow from "S is there".
//
// Bound by the exponentials: 128 x 128 weights at 16 a clock are 1024 clocks, its two products 1024 on the tensor cores.
#pragma once

#include "paged_work.cuh"

namespace b200ipc {

constexpr int kWideRows = 256;
constexpr int kWideTile = 128;   // positions
constexpr int kWideStages = 5;   // K or V tiles
constexpr int kWideQueue = 4;    // items handed out ahead
constexpr int kWideThreads = 384;  // three warpgroups
constexpr int kWideRegsSoftmax = 224, kWideRegsRest = 56;  // 256 x 208 + 128 x 88 = 384 x 168, what the launch has
constexpr int kWideTileBytes = kWideTile * kAttnD * 2;  // also of 128 rows of Q
constexpr size_t kWideSmem = 1024 + size_t(kWideStages + 2) * kWideTileBytes;
constexpr int kWideStart = 192;  // what an item's start and end cost, in positions
constexpr int kWideLeast = 384;  // a span is at least so long: more than kWideStart + a tile, so that every cut leaves a tile on both sides
constexpr float kWideSlack = 8.f;

struct WideCut {
  const PagedArgs& a;
  __device__ __forceinline__ bool takes(const Request& r) const { return r.n > 0 && r.n * a.group > a.narrow_rows; }
  __device__ __forceinline__ int items(const Request& r) const { return (r.n * a.group + kWideRows - 1) / kWideRows; }
  // positions that the rows below `row` of the request see
  __device__ __forceinline__ int seen(const Request& r, int rows) const {
    return rows <= 0 ? 0 : max(0, r.len - r.n + (min(rows, r.n * a.group) - 1) / a.group + 1);
  }
  __device__ __forceinline__ int tiles(const Request& r, int item) const { return (seen(r, (item + 1) * kWideRows) + kWideTile - 1) / kWideTile; }
  // Length of the first `t` items of a head, in positions x group: item u sees max(len - n, 0) + (u + 1) * 256 / group positions or a few less.
  __device__ __forceinline__ int64_t before(const Request& r, int64_t t) const {
    return t * (int64_t(max(0, r.len - r.n)) + kWideStart) * a.group + (kWideRows / 2) * t * (t + 1);
  }
  __device__ __forceinline__ int64_t length(const Request& r) const { return takes(r) ? a.hkv * before(r, items(r)) : 0; }
  __device__ __forceinline__ int4 place(const Mark& m) const {
    if (m.request >= a.requests) return make_int4(a.requests, 0, 0, 0);
    const Request r = request_at(a, m.request);
    const int n = items(r);
    const int64_t per = before(r, n);
    const int h = int(m.offset / per);
    const int64_t rest = m.offset - h * per;
    int lo = 0, hi = n;  // the last item that begins at or before `rest`
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before(r, mid) <= rest) lo = mid;
      else hi = mid;
    }
    const int64_t in = rest - before(r, lo) - int64_t(kWideStart) * a.group;
    const int t = in <= 0 ? 0 : int((in + int64_t(kWideTile / 2) * a.group) / (int64_t(kWideTile) * a.group));
    const int all = tiles(r, lo);
    if (t >= all && all > 0) {  // rounded to its end: the next item
      if (lo + 1 < n) return make_int4(m.request, h * n + lo + 1, 0, 0);
      if (h + 1 < a.hkv) return make_int4(m.request, (h + 1) * n, 0, 0);
      return make_int4(m.request + 1, 0, 0, 0);
    }
    return make_int4(m.request, h * n + lo, min(t, max(all - 1, 0)), 0);
  }
};

// The part of an item that lies in a span, as the scheduling warp hands it to the others.
struct WideItem {
  int valid;
  int request, h;       // KV head
  int first, n, len;    // the request's first row of q, its new tokens, its tokens in the cache
  int row0, rows;       // rows of the item within the request
  int t0, t1, whole;    // tiles of positions; whether these are all
  int count[2];         // tiles of positions from t0 on that accumulator tile w looks at
};

// The span's items one after the other.
struct WideWalk {
  const PagedArgs& a;
  const WideCut cut;
  const int4 last;
  Window win;
  int i, number, t0;
  __device__ __forceinline__ WideWalk(const PagedArgs& args, const int4& first, const int4& end) : a(args), cut{args}, last(end), i(first.x), number(first.y), t0(first.z) {}
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
    if (i >= a.requests || i > last.x || (i == last.x && (number > last.y || (number == last.y && t0 >= last.z)))) return x;
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
    x.t1 = i == last.x && number == last.y ? last.z : tiles;
    x.whole = t0 == 0 && x.t1 == tiles;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int see = x.rows > w * 128 ? cut.seen(r, x.row0 + min(x.rows, (w + 1) * 128)) : 0;
      x.count[w] = max(0, min((see + kWideTile - 1) / kWideTile, x.t1) - x.t0);
    }
    t0 = 0;
    if (++number == a.hkv * n) {
      number = 0;
      ++i;
    }
    return x;
  }
};

__device__ __forceinline__ void tmem_st_32cols(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
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

template <typename T>
__global__ void __launch_bounds__(kWideThreads, 1) paged_wide_kernel(const __grid_constant__ PagedArgs args) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t kv_full[kWideStages], kv_empty[kWideStages], q_ready[2], s_full[2], p_ready[2], o_full[2], item_full[kWideQueue], item_empty[kWideQueue], mma_done;
  __shared__ WideItem s_items[kWideQueue];
  __shared__ Mark s_marks[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  unsigned char* q_smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* ring = q_smem + 2 * kWideTileBytes;
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = int(threadIdx.x & 31);
  volatile int* abort_flag = &s_abort;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kWideStages; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&q_ready[w], 128);
      mbar_init(&s_full[w], 1);
      mbar_init(&p_ready[w], 128);
      mbar_init(&o_full[w], 1);
    }
    for (int i = 0; i < kWideQueue; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 10);
    }
    mbar_init(&mma_done, 1);
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
  find_span<kWideThreads>(args, [&](const Request& r) { return cut.length(r); }, int64_t(kWideLeast) * args.group, s_marks);
  tc_fence_after_sync();
  const uint32_t tmem = s_tmem;
  const int4 first = cut.place(s_marks[0]), last = cut.place(s_marks[1]);
  if (threadIdx.x == 0) {
    args.starts[blockIdx.x] = first;
    if (blockIdx.x == gridDim.x - 1) args.starts[gridDim.x] = last;
  }
  lead<T>(args);
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!*abort_flag) mbar_wait_long(bar, parity, abort_flag, kPagedTimeoutNs);
  };

  // The items as a role sees them: one in hand at a time, given back when it is done with.
  uint32_t item_at = 0, item_ph = 0;
  auto take = [&]() {  // nullptr behind the last one
    wait(&item_full[item_at], item_ph);
    const WideItem* x = &s_items[item_at];
    return x->valid && !__any_sync(0xffffffffu, *abort_flag) ? x : nullptr;
  };
  auto give_back = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[item_at]);
    if (++item_at == kWideQueue) {
      item_at = 0;
      item_ph ^= 1u;
    }
  };
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWideRegsSoftmax));
    // ---- softmax: thread = row of tile w ------------------------------------------------------------------------------------
    const int w = warp >> 2, row = (warp & 3) * 32 + lane, G = args.group;
    const uint32_t lane_base = tmem + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t s_addr = lane_base + uint32_t(w) * 128u, o_addr = lane_base + 256u + uint32_t(w) * 128u;
    unsigned char* q_row = q_smem + w * kWideTileBytes + row * 128;
    uint32_t ph_s = 0, ph_o = 0, ring_at = 0, ring_ph = 0;  // the ring position of the item's first K tile
    auto load_q = [&](const WideItem* x) {
      if (x == nullptr || x->rows <= w * 128) return;
      const int at = x->row0 + w * 128 + row, j = at / G;
      uint4 v[16];
      if (w * 128 + row < x->rows) {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(args.q) + int64_t(x->first + j) * args.row_stride + (int64_t(x->h) * G + (at - j * G)) * kAttnD);
#pragma unroll
        for (int c = 0; c < 16; ++c) v[c] = src[c];
      } else {
#pragma unroll
        for (int c = 0; c < 16; ++c) v[c] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int c = 0; c < 16; ++c) *reinterpret_cast<uint4*>(q_row + (c >> 3) * (kWideTileBytes / 2) + (((c & 7) ^ (row & 7)) << 4)) = v[c];
      fence_async_smem();
      mbar_arrive(&q_ready[w]);
    };
    const WideItem* x = take();
    load_q(x);
    while (x != nullptr) {
      // fields that are needed after the item has been given back
      const int n = x->t1 - x->t0, t0 = x->t0, len = x->len, h = x->h, first_row = x->first;
      const bool whole = x->whole != 0;
      const WideItem* following;
      if (x->rows > w * 128) {
        const int at = x->row0 + w * 128 + row, j = at / G;
        const bool exists = w * 128 + row < x->rows;
        const int limit = exists ? len - x->n + j + 1 : 0;  // positions that this row sees
        const int count = x->count[w], clears = w == 0 ? 0 : x->count[0];  // from which tile on this one uses V first
        float ref = -INFINITY, sum = 0;  // the maximum that the weights are taken against (log2 domain)
        for (int t = 0; t < count; ++t) {
          const int p0 = (t0 + t) * kWideTile;
          wait(&s_full[w], ph_s);
          ph_s ^= 1u;
          tc_fence_after_sync();
          float s[kWideTile];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld_32cols(s_addr + uint32_t(c) * 32u, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * c]));
          tmem_ld_wait();
          if (__any_sync(0xffffffffu, limit < p0 + kWideTile)) {
#pragma unroll
            for (int c = 0; c < kWideTile; ++c)
              if (p0 + c >= limit) s[c] = -INFINITY;
          }
          float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
          for (int c = 4; c < kWideTile; c += 4)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], s[c + e]);
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * args.scale_log2;
          if (__any_sync(0xffffffffu, top > ref + kWideSlack)) {
            const float now = fmaxf(ref, top);
            if (t > 0) {
              const float f = now == -INFINITY ? 1.f : exp2_fast(ref - now);
              sum *= f;
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                uint32_t o[32];
                tmem_ld_32cols(o_addr + uint32_t(c) * 32u, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st_32cols(o_addr + uint32_t(c) * 32u, o);
              }
            }
            ref = now;
          }
          const float shift = ref == -INFINITY ? 0.f : -ref;
          float part[4] = {0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t p[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float a = exp2_fast(fmaf(s[64 * c + 2 * e], args.scale_log2, shift)), b = exp2_fast(fmaf(s[64 * c + 2 * e + 1], args.scale_log2, shift));
              part[2 * (e & 1)] += a;
              part[2 * (e & 1) + 1] += b;
              p[e] = pack2<T>(a, b);
            }
            tmem_st_32cols(s_addr + uint32_t(c) * 32u, p);
          }
          sum += (part[0] + part[1]) + (part[2] + part[3]);
          // Values of positions that do not exist count as zero (a weight of zero would not do: they may be NaN).  Whichever tile uses
          // this V tile first clears them.
          if (p0 + kWideTile > len && t >= clears) {
            const uint32_t v_at = ring_at + uint32_t(2 * t + 1);
            const uint32_t v_st = v_at % kWideStages, v_ph = ring_ph ^ ((v_at / kWideStages) & 1u);
            wait(&kv_full[v_st], v_ph);
            if (p0 + row >= len) {
              unsigned char* v = ring + v_st * kWideTileBytes + row * 128;
#pragma unroll
              for (int c = 0; c < 16; ++c) *reinterpret_cast<uint4*>(v + (c >> 3) * (kWideTileBytes / 2) + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
            }
            fence_async_smem();
          }
          tmem_st_wait();
          tc_fence_before_sync();
          mbar_arrive(&p_ready[w]);
        }
        give_back();
        following = take();
        load_q(following);  // S of this item is complete, so Q is free
        if (count > 0) {
          wait(&o_full[w], ph_o);
          ph_o ^= 1u;
          tc_fence_after_sync();
        }
        if (whole) {
          const float inv = sum == 0 ? 0.f : 1 / sum;  // a row that sees nothing
          T* dst = static_cast<T*>(args.out) + (int64_t(first_row + j) * args.hq + int64_t(h) * G + (at - j * G)) * kAttnD;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t o[32];
            if (count > 0) {
              tmem_ld_32cols(o_addr + uint32_t(c) * 32u, o);
              tmem_ld_wait();
            }
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(sum == 0 ? 0.f : __uint_as_float(o[e]) * inv);
            if (exists) {
#pragma unroll
              for (int e = 0; e < 32; e += 8) {
                auto pair = [&](int k) { return pack2<T>(__uint_as_float(o[e + 2 * k]), __uint_as_float(o[e + 2 * k + 1])); };
                *reinterpret_cast<uint4*>(dst + 32 * c + e) = make_uint4(pair(0), pair(1), pair(2), pair(3));
              }
            }
          }
        } else {
          float* piece = Piece<kWideRows>::slot(args, int(blockIdx.x), t0 > 0 ? 0 : 1);
          const int r = w * 128 + row;
          if (exists) *reinterpret_cast<float2*>(piece + 2 * r) = make_float2(ref, sum);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t o[32];
            if (count > 0) {
              tmem_ld_32cols(o_addr + uint32_t(c) * 32u, o);
              tmem_ld_wait();
            }
            if (exists) {
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                const bool some = count > 0;
                *reinterpret_cast<uint4*>(piece + 2 * kWideRows + size_t(r) * kAttnD + 32 * c + e) =
                    some ? make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]) : make_uint4(0, 0, 0, 0);
              }
            }
          }
        }
        tc_fence_before_sync();  // O may be written again once this thread's next weights are there
      } else {
        give_back();
        following = take();
        load_q(following);
      }
      const uint32_t moved = ring_at + uint32_t(2 * n);
      ring_ph ^= (moved / kWideStages) & 1u;
      ring_at = moved % kWideStages;
      x = following;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWideRegsRest));
    if (warp == 8) {
      // ---- the stream: lane l loads box l / 2 of a tile, left or right half of the dimensions --------------------------------
      const int box = min(args.page, 64), boxes = kWideTile / box, per_page = args.page / box;
      const int sub = lane >> 1, half = lane & 1;
      const int64_t outside = args.pages * args.hkv * args.page;
      uint32_t st = 0, ph = 0;
      int issued = 0;
      for (const WideItem* x = take(); x != nullptr; x = take()) {
        const int* table = args.table + int64_t(x->request) * args.width;
        const int len = x->len, h = x->h, pages = (len + args.page - 1) / args.page, t1 = x->t1;
        int base = -64, entry = 0;
        for (int t = x->t0; t < t1; ++t) {
          const int b = t * boxes + sub, p = b / per_page, offset = (b - p * per_page) * box;
          const int p_first = t * boxes / per_page;
          if (p_first < base || (t * boxes + boxes - 1) / per_page >= base + 32) {
            base = p_first;
            entry = base + lane < pages ? table[base + lane] : -1;
          }
          const int64_t id = __shfl_sync(0xffffffffu, entry, min(31, p - base));
          const int n = min(boxes, (len - t * kWideTile + box - 1) / box);  // boxes that hold positions of the request
          const int row = int(id >= 0 && id < args.pages ? (id * args.hkv + h) * args.page + offset : outside);
  #pragma unroll
          for (int value = 0; value < 2; ++value) {
            wait(&kv_empty[st], ph ^ 1u);
            if (!__any_sync(0xffffffffu, *abort_flag)) {
              if (lane == 0) mbar_expect_tx(&kv_full[st], uint32_t(n * box) * kAttnD * 2u);
              __syncwarp();
              if (sub < n) tma_load_2d(ring + st * kWideTileBytes + half * (kWideTileBytes / 2) + sub * box * 128, value ? &args.tma_v : &args.tma_k, &kv_full[st], half * 64, row);
              ++issued;
              if (++st == kWideStages) {
                st = 0;
                ph ^= 1u;
              }
            }
          }
        }
        give_back();
      }
      const uint64_t since = globaltimer_ns();
      for (int back = 1; back <= min(issued, kWideStages); ++back)
        mbar_drain(&kv_full[(issued - back) % kWideStages], uint32_t((issued - back) / kWideStages) & 1u, since);
    } else if (warp == 9) {
      // ---- the products ----------------------------------------------------------------------------------------------------
      const uint32_t idesc_s = make_idesc<T>(128, kWideTile), idesc_o = make_idesc<T>(128, kAttnD) | (1u << 16);
      const uint32_t q_addr = smem_u32(q_smem), ring_addr = smem_u32(ring);
      uint32_t ring_at = 0, ring_ph = 0;  // the next tile that has not been waited for
      uint32_t ph_q[2] = {0, 0}, ph_p[2] = {0, 0};
      auto next_tile = [&]() {
        wait(&kv_full[ring_at], ring_ph);
        const uint32_t st = ring_at;
        if (++ring_at == kWideStages) {
          ring_at = 0;
          ring_ph ^= 1u;
        }
        return st;
      };
      // 64 columns of a K-major tile are one block of it, 16 of them 32 bytes of its rows; descriptors count in 16 bytes
      const uint64_t q_desc = make_sw128_kmajor_desc(q_addr), k_desc = make_sw128_kmajor_desc(ring_addr), v_desc = make_sw128_nmajor_desc(ring_addr);
      constexpr uint64_t kTileStep = kWideTileBytes >> 4, kBlockStep = kWideTileBytes >> 5;
      auto scores = [&](int w, uint32_t k_st) {
        tc_fence_after_sync();
        if (elect_one()) {
          const uint64_t a = q_desc + uint64_t(w) * kTileStep, b = k_desc + uint64_t(k_st) * kTileStep;
  #pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint64_t at = uint64_t(k >> 2) * kBlockStep + uint64_t(k & 3) * 2u;
            umma_f16(tmem + uint32_t(w) * 128u, a + at, b + at, idesc_s, k > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[w]);
        }
        __syncwarp();
      };
      auto outputs = [&](int w, uint32_t v_st, bool fresh) {
        wait(&p_ready[w], ph_p[w]);
        ph_p[w] ^= 1u;
        tc_fence_after_sync();
        if (elect_one()) {
          const uint64_t b = v_desc + uint64_t(v_st) * kTileStep;
  #pragma unroll
          for (int k = 0; k < kWideTile / 16; ++k)  // 16 positions: 8 columns of P, 2048 bytes of V
            umma_f16_ts(tmem + 256u + uint32_t(w) * 128u, tmem + uint32_t(w) * 128u + uint32_t(k) * 8u, b + uint64_t(k) * 128u, idesc_o, !fresh || k > 0 ? 1u : 0u);
        }
        __syncwarp();
      };
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) umma_commit(bar);
        __syncwarp();
      };
      for (const WideItem* x = take(); x != nullptr; x = take()) {
        const int n = x->t1 - x->t0, count[2] = {x->count[0], x->count[1]};
  #pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (x->rows > w * 128) {
            wait(&q_ready[w], ph_q[w]);
            ph_q[w] ^= 1u;
          }
        }
        if (n > 0) {
          const uint32_t st = next_tile();
  #pragma unroll
          for (int w = 0; w < 2; ++w)
            if (count[w] > 0) scores(w, st);
          commit(&kv_empty[st]);
        }
        for (int j = 0; j < n; ++j) {
          const uint32_t v_st = next_tile(), k_st = j + 1 < n ? next_tile() : 0u;
  #pragma unroll
          for (int w = 0; w < 2; ++w) {
            if (j < count[w]) outputs(w, v_st, j == 0);
            if (w == 0 ? count[1] <= j : j < count[1]) commit(&kv_empty[v_st]);  // its last reader
            if (j + 1 < count[w]) scores(w, k_st);
            else if (j + 1 == count[w]) commit(&o_full[w]);
          }
          if (j + 1 < n) commit(&kv_empty[k_st]);
        }
        give_back();
      }
      commit(&mma_done);
      mbar_drain(&mma_done, 0, globaltimer_ns());
    } else if (warp == 10) {
      // ---- the items -----------------------------------------------------------------------------------------------------------
      WideWalk walk(args, first, last);
      for (bool more = true; more;) {
        const WideItem x = walk.next();
        wait(&item_empty[item_at], item_ph ^ 1u);
        more = x.valid && !__any_sync(0xffffffffu, *abort_flag);
        if (lane == 0) {
          s_items[item_at] = x;
          mbar_arrive(&item_full[item_at]);
        }
        __syncwarp();
        if (++item_at == kWideQueue) {
          item_at = 0;
          item_ph ^= 1u;
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 9) tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && *abort_flag) *args.status = 1;
}

constexpr int kWideJoin = 4;  // warps of a row
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_wide_join_kernel(const __grid_constant__ PagedArgs args, int spans) {
  pdl_launch_dependents();
  pdl_wait();
  join_rows<T, kWideRows, kWideJoin>(args, spans, [&](const int4& mark, int row) -> T* {
    const WideCut cut{args};
    const Request r = request_at(args, mark.x);
    const int n = cut.items(r), h = mark.y / n, at = (mark.y - h * n) * kWideRows + row;
    if (at >= r.n * args.group) return nullptr;
    const int j = at / args.group;
    return static_cast<T*>(args.out) + (int64_t(r.row0 + j) * args.hq + int64_t(h) * args.group + (at - j * args.group)) * kAttnD;
  });
}

}  // namespace b200ipc
