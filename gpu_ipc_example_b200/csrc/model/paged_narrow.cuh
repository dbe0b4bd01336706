// Attention over a paged cache for requests with few rows: up to 16 of (new tokens x query heads of a KV head).  Single tokens of a
// decoding server, a few drafts behind them.
//
// Bound by memory: every position of a request is 512 bytes of K and V per KV head and read once for all of the item's rows.  One warp
// streams the pages by TMA (128-byte swizzle) into a ring of four stages of 64 positions, 128 KB in flight per SM (six
// are no faster, and leave no room for the next kernel's CTAs to come up); a page that the cache
// does not have is a box outside of the tensor, which reads zeros.  Eight warps compute with mma.sync (m16n8k16): 16 rows cannot fill
// tcgen05's 128.  Warps 0-3 take the tiles in even stages, 4-7 those in odd ones (always the same stages: a wait for a stage's next round
// must come from who has seen the round before, as copies may land out of order), 16 positions of a tile each.  Scores, maxima, sums
// and outputs are fp32; the weights are rounded to 16 bits for the second product, as the tensor cores take them.
//
// 16 requests of up to 32768 tokens, two KV heads: 290 MB in 53 us, 5.4 TB/s over the launch; 32 of 2048, one KV head: 33.7 MB in 15.5 us, of which
// 5.1 would be memory's: 4 pass until the first tile is there (lengths, span, table, copy, each a round to memory behind the other), 3 at
// the end (pieces out, the last CTA's reads, its rows out).
#pragma once

#include "paged_work.cuh"

namespace b200ipc {

constexpr int kNarRows = 16;
constexpr int kNarTile = 64;     // positions
constexpr int kNarStages = 4;    // even: a stage belongs to one half of the warps
constexpr int kNarWarps = 8;     // that compute; then the stream's and the walking one
constexpr int kNarThreads = (kNarWarps + 2) * 32;
constexpr int kNarTileBytes = kNarTile * kAttnD * 2;  // of K or V
constexpr int kNarORow = kAttnD + 4;                  // floats of a row of the merge buffer
constexpr size_t kNarSmem = 1024 + size_t(kNarStages) * 2 * kNarTileBytes + size_t(kNarWarps) * 8 * kNarORow * 4;
constexpr int kNarStart = 1;     // what an item's start and end cost, in tiles
constexpr int kNarLeast = 4;     // a span is at least so long: more than kNarStart, so that every cut leaves a tile on both sides

struct NarrowItem {
  int valid;
  int request, h;       // KV head
  int first, n, len;    // the request's first row of q, its new tokens, its tokens in the cache
  int t0, t1;           // tiles of positions
  int from, pieces;     // the span that the item begins in, and in how many it is
};

struct NarrowCut {
  const PagedArgs& a;
  __device__ __forceinline__ bool takes(const Request& r) const { return r.n > 0 && r.n * a.group <= kNarRows; }
  __device__ __forceinline__ int tiles(const Request& r) const { return (r.len + kNarTile - 1) / kNarTile; }
  __device__ __forceinline__ uint64_t length(const Request& r) const { return takes(r) ? uint64_t(a.hkv) * uint32_t(kNarStart + tiles(r)) : 0; }
  __device__ __forceinline__ Start place(const Request& r, int request, uint64_t offset) const {
    const uint32_t per = uint32_t(kNarStart + tiles(r));
    const int h = int(divide(offset, per));
    return Start{request, h, max(0, int(offset - uint64_t(h) * per) - kNarStart), h, 0, r.n * a.group, r, uint64_t(h) * per};  // + the request's
  }
};

__device__ __forceinline__ void nar_ldmatrix(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void nar_ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kNarThreads, 1) paged_narrow_kernel(const __grid_constant__ PagedArgs args) {
  extern __shared__ unsigned char smem_raw[];
  using Items = Queue<NarrowItem, kNarWarps + 1>;
  __shared__ Items s_queue;
  __shared__ uint64_t full[kNarStages], empty[kNarStages];
  __shared__ int s_abort;
  __shared__ uint64_t s_sum[kNarThreads / 32];
  __shared__ Start s_span[2];
  __shared__ Axis s_axis;
  __shared__ int s_last;
  __shared__ float2 s_ml[kNarWarps][8];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_o = reinterpret_cast<float*>(ring + kNarStages * 2 * kNarTileBytes);  // [8 warps][8 rows][kNarORow]
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = int(threadIdx.x & 31);
  volatile int* abort_flag = &s_abort;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kNarStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    s_queue.init();
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  const NarrowCut cut{args};
  find_span<kNarThreads>(
      args, [&](const Request& r) { return cut.length(r); }, [&](const Request& r, int i, uint64_t o) { return cut.place(r, i, o); }, kNarLeast, s_sum, s_span, &s_axis);
  __syncthreads();
  QueueEnd<Items, NarrowItem> items{s_queue, abort_flag, args.timeout_ns};

  if (warp == kNarWarps + 1) {
    // ---- the walk ------------------------------------------------------------------------------------------------------------
    const Start first = s_span[0], last = s_span[1];
    Window win;
    Request r = first.r;
    int i = first.request, h = first.number, t0 = first.tile;
    for (;;) {
      NarrowItem x{};
      if (i < args.requests && !(i > last.request || (i == last.request && (h > last.number || (h == last.number && t0 >= last.tile))))) {
        const int tiles = cut.tiles(r), t1 = i == last.request && h == last.number ? last.tile : tiles;
        x = NarrowItem{1, i, h, r.row0, r.n, r.len, t0, t1, int(blockIdx.x), 1};
        if (t0 > 0 || t1 < tiles) {  // its first tile may be looked for up to kNarStart behind its beginning
          const uint64_t origin = t0 > 0 ? first.origin : last.origin;
          x.from = span_of(s_axis, origin + kNarStart);
          x.pieces = span_of(s_axis, origin + kNarStart + uint32_t(tiles) - 1) - x.from + 1;
        }
      }
      if (!items.put(x)) break;
      t0 = 0;
      if (++h == args.hkv) {
        h = 0;
        i = win.next(args, i + 1, [&](const Request& y) { return cut.takes(y); });
        if (i < args.requests) r = win.get(i);
      }
    }
  } else if (warp == kNarWarps) {
    // ---- the stream: lane l knows where box l of a tile is; K and V, left and right half of the dimensions --------------------
    const int box_log = min(args.page_log, 6), box = 1 << box_log, boxes_log = 6 - box_log, boxes = 1 << boxes_log, per_page = args.page_log - box_log;
    uint32_t st = 0, ph = 0;
    int issued = 0;
    for (const NarrowItem* x = items.take(); x != nullptr; x = items.take()) {
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
        const int n = min(boxes, (len - t * kNarTile + box - 1) >> box_log);  // boxes that hold positions of the request
        items.wait_warp(&empty[st], ph ^ 1u);
        if (__any_sync(0xffffffffu, *abort_flag)) break;
        const int sent = args.mute && blockIdx.x == 0 && issued == 0 ? 0 : n;
        if (lane == 0 && sent > 0) mbar_expect_tx(&full[st], uint32_t(n << box_log) * kAttnD * 4u);
        __syncwarp();
        unsigned char* dst = ring + st * 2 * kNarTileBytes;
        for (int k = 0; k < sent; ++k, dst += box * 128) {
          const int row = __shfl_sync(0xffffffffu, at, k);
          if (elect_one()) {
            tma_load_2d(dst, &args.tma_k, &full[st], 0, row);
            tma_load_2d(dst + kNarTileBytes / 2, &args.tma_k, &full[st], 64, row);
            tma_load_2d(dst + kNarTileBytes, &args.tma_v, &full[st], 0, row);
            tma_load_2d(dst + kNarTileBytes + kNarTileBytes / 2, &args.tma_v, &full[st], 64, row);
          }
          __syncwarp();
        }
        ++issued;
        if (++st == kNarStages) {
          st = 0;
          ph ^= 1u;
        }
      }
      items.give_back();
    }
    // copies in flight land before the CTA leaves
    const uint64_t since = globaltimer_ns();
    for (int back = 1; back <= min(issued, kNarStages); ++back)
      mbar_drain(&full[(issued - back) % kNarStages], uint32_t((issued - back) / kNarStages) & 1u, since);
  } else {
    // ---- the arithmetic ----------------------------------------------------------------------------------------------------
    const int side = warp >> 2, r8 = lane >> 2, c = lane & 3, G = args.group, at = (warp & 3) * 16;  // positions of a tile: at .. at + 15
    const uint32_t ring_addr = smem_u32(ring);
    const uint32_t k_row = uint32_t(at + ((lane >> 4) & 1) * 8 + (lane & 7)), k_chunk = (lane >> 3) & 1;
    const uint32_t v_row = uint32_t(at + ((lane >> 3) & 1) * 8 + (lane & 7)), v_chunk = (lane >> 4) & 1;
    auto chunk_addr = [](uint32_t tile, uint32_t pos, uint32_t chunk) {
      return tile + (chunk >> 3) * (kNarTileBytes / 2) + pos * 128 + (((chunk & 7) ^ (pos & 7)) << 4);
    };
    uint32_t st = 0, ph = 0;
    uint32_t qa[8][4];
    // this lane's two rows of an item, r8 and r8 + 8
    auto load_q = [&](const NarrowItem* x) {
      const int nrows = x->n * G;
      auto row_of = [&](int row) {
        const int j = row / G;
        return reinterpret_cast<const uint32_t*>(static_cast<const T*>(args.q) + int64_t(x->first + j) * args.row_stride + (int64_t(x->h) * G + (row - j * G)) * kAttnD);
      };
      const bool a = r8 < nrows, b = r8 + 8 < nrows;
      const uint32_t *pa = row_of(a ? r8 : 0), *pb = row_of(b ? r8 + 8 : 0);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        qa[k][0] = a ? pa[8 * k + c] : 0u;
        qa[k][1] = b ? pb[8 * k + c] : 0u;
        qa[k][2] = a ? pa[8 * k + 4 + c] : 0u;
        qa[k][3] = b ? pb[8 * k + 4 + c] : 0u;
      }
    };
    const NarrowItem* x = items.take();
    if (x != nullptr) load_q(x);
    while (x != nullptr) {
      const int nrows = x->n * G, len = x->len, t0 = x->t0, t1 = x->t1, h = x->h, first_row = x->first;
      const int from = x->from, pieces = x->pieces;
      const bool whole = pieces == 1;
      // positions that the rows see
      const int all_see = len - x->n + 1;
      const int la = r8 < nrows ? all_see + r8 / G : 0, lb = r8 + 8 < nrows ? all_see + (r8 + 8) / G : 0;
      float ma = -INFINITY, mb = -INFINITY, sa = 0, sb = 0;
      float o[16][4];
#pragma unroll
      for (int d = 0; d < 16; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0;
      for (int t = t0; t < t1; ++t) {
        if (int(st & 1u) == side) {
          items.wait_warp(&full[st], ph);
          const uint32_t kt = ring_addr + st * 2 * kNarTileBytes, vt = kt + kNarTileBytes;
          const int pos = t * kNarTile + at;
          if (pos < len) {
            float s[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}}, s2[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};  // two chains: half as long
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              uint32_t kf[4];
              nar_ldmatrix(kf, chunk_addr(kt, k_row, 2 * k + k_chunk));
              mma_16816<T>(k & 1 ? s2[0] : s[0], qa[k][0], qa[k][1], qa[k][2], qa[k][3], kf[0], kf[1]);
              mma_16816<T>(k & 1 ? s2[1] : s[1], qa[k][0], qa[k][1], qa[k][2], qa[k][3], kf[2], kf[3]);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[j][e] = (s[j][e] + s2[j][e]) * args.scale_log2;
            if (pos + 16 > all_see) {
#pragma unroll
              for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int p = pos + 8 * j + 2 * c + e;
                  if (p >= la) s[j][e] = -INFINITY;
                  if (p >= lb) s[j][2 + e] = -INFINITY;
                }
            }
            float xa = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])), xb = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
#pragma unroll
            for (int d = 1; d < 4; d <<= 1) {
              xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, d));
              xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, d));
            }
            if (__any_sync(0xffffffffu, xa > ma || xb > mb)) {
              const float na = fmaxf(ma, xa), nb = fmaxf(mb, xb);
              const float ca = na == -INFINITY ? 1.f : exp2_fast(ma - na), cb = nb == -INFINITY ? 1.f : exp2_fast(mb - nb);
              ma = na;
              mb = nb;
              sa *= ca;
              sb *= cb;
#pragma unroll
              for (int d = 0; d < 16; ++d) {
                o[d][0] *= ca; o[d][1] *= ca; o[d][2] *= cb; o[d][3] *= cb;
              }
            }
            const float ua = ma == -INFINITY ? 0.f : ma, ub = mb == -INFINITY ? 0.f : mb;
            uint32_t pw[4];  // the weights as the next product's left operand
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float p0 = exp2_fast(s[j][0] - ua), p1 = exp2_fast(s[j][1] - ua), p2 = exp2_fast(s[j][2] - ub), p3 = exp2_fast(s[j][3] - ub);
              sa += p0 + p1;
              sb += p2 + p3;
              pw[2 * j] = pack2<T>(p0, p1);
              pw[2 * j + 1] = pack2<T>(p2, p3);
            }
            // values of positions that do not exist count as zero (a weight of zero would not do: they may be NaN)
            uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
            if (pos + 16 > len) {
              const int left = len - pos - 2 * c;
              keep0 = left <= 0 ? 0u : left == 1 ? 0xffffu : 0xffffffffu;
              keep1 = left <= 8 ? 0u : left == 9 ? 0xffffu : 0xffffffffu;
            }
#pragma unroll
            for (int d = 0; d < 8; ++d) {
              uint32_t vf[4];
              nar_ldmatrix_trans(vf, chunk_addr(vt, v_row, 2 * d + v_chunk));
              mma_16816<T>(o[2 * d], pw[0], pw[1], pw[2], pw[3], vf[0] & keep0, vf[1] & keep1);
              mma_16816<T>(o[2 * d + 1], pw[0], pw[1], pw[2], pw[3], vf[2] & keep0, vf[3] & keep1);
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[st]);
        }
        if (++st == kNarStages) {
          st = 0;
          ph ^= 1u;
        }
      }
      items.give_back();
      x = items.take();
      if (x != nullptr) load_q(x);  // on its way while this item is put together
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        sa += __shfl_xor_sync(0xffffffffu, sa, d);
        sb += __shfl_xor_sync(0xffffffffu, sb, d);
      }
      // ---- the warps' parts of rows 0 - 7, then of 8 - 15, are added: a warp per row, four dimensions a lane ------------
      float* piece = whole ? nullptr : Piece<kNarRows>::slot(args, blockIdx.x, t0 > 0 ? 0 : 1);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (half * 8 >= nrows) break;
        float* mine = s_o + (warp * 8 + r8) * kNarORow;
#pragma unroll
        for (int d = 0; d < 16; ++d) *reinterpret_cast<float2*>(mine + 8 * d + 2 * c) = make_float2(o[d][2 * half], o[d][2 * half + 1]);
        if (c == 0) s_ml[warp][r8] = half == 0 ? make_float2(ma, sa) : make_float2(mb, sb);
        meet<kNarWarps * 32>();
        const int row = half * 8 + warp;
        if (row < nrows) {
          float2 ml[kNarWarps];
          float m = -INFINITY, l = 0;
#pragma unroll
          for (int w = 0; w < kNarWarps; ++w) {
            ml[w] = s_ml[w][warp];
            m = fmaxf(m, ml[w].x);
          }
          const float u = m == -INFINITY ? 0.f : m;
          float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
          for (int w = 0; w < kNarWarps; ++w) {
            const float f = exp2_fast(ml[w].x - u);
            const float4 y = *reinterpret_cast<const float4*>(s_o + (w * 8 + warp) * kNarORow + lane * 4);
            l += ml[w].y * f;
            v = make_float4(v.x + y.x * f, v.y + y.y * f, v.z + y.z * f, v.w + y.w * f);
          }
          if (whole) {
            const int j = row / G;
            const float4 y = divided(v, l, all_see + j > 0);
            T* dst = static_cast<T*>(args.out) + (int64_t(first_row + j) * args.hq + int64_t(h) * G + (row - j * G)) * kAttnD + lane * 4;
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(y.x, y.y), pack2<T>(y.z, y.w));
          } else {
            if (lane == 0) *reinterpret_cast<float2*>(piece + 2 * row) = make_float2(m, l);
            *reinterpret_cast<float4*>(piece + 2 * kNarRows + row * kAttnD + lane * 4) = v;
          }
        }
        meet<kNarWarps * 32>();
      }
      if (!whole) {  // who is last puts the item together
        if (threadIdx.x == 0) {  // behind the barrier: what it releases and acquires is the other warps' as well
          unsigned before;
          asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(args.arrived + from) : "memory");
          s_last = before == unsigned(pieces - 1);
          if (s_last) args.arrived[from] = 0;  // for the next call
        }
        meet<kNarWarps * 32>();
        if (s_last) {
          for (int row = warp; row < nrows; row += kNarWarps) {
            Joined sum;
#pragma unroll 4
            for (int n = 0; n < pieces; ++n) {
              const float* p = Piece<kNarRows>::slot(args, from + n, n == 0 ? 1 : 0);
              sum.add(__ldcg(reinterpret_cast<const float2*>(p + 2 * row)), __ldcg(reinterpret_cast<const float4*>(p + 2 * kNarRows + row * kAttnD + lane * 4)));
            }
            const int j = row / G;
            const float4 y = divided(sum.o, sum.l, all_see + j > 0);
            T* dst = static_cast<T*>(args.out) + (int64_t(first_row + j) * args.hq + int64_t(h) * G + (row - j * G)) * kAttnD + lane * 4;
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(y.x, y.y), pack2<T>(y.z, y.w));
          }
        }
      }
    }
    while (!meet<kNarWarps * 32>(true)) {
    }
  }
  zero_tail<T>(args);
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) atomicOr(args.status, kPagedGaveUp);
}

}  // namespace b200ipc
