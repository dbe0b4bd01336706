// Attention over a paged cache for requests with few rows: up to 64 of (new tokens x query heads of a KV head).  Single tokens of a decoding
// server, drafts behind them, short prompts.
//
// Bound by memory: every position of a request is 512 bytes of K and V per KV head and read once for all of the item's rows.  One thread
// per box streams the pages by TMA (128-byte swizzle) into a ring of six stages of 64 positions, 192 KB in flight per SM; a page that the cache
// does not have is a box outside of the tensor, which reads zeros.  Eight warps compute with mma.sync (m16n8k16): at most 64 rows
// cannot fill tcgen05's 128, and its accumulators would have to be fetched back for every 64 positions.  Warps 0-3 take the tiles in even
// stages, 4-7 those in odd ones (always the same stages: a wait for a stage's next round must come from who has seen the round before, as
// copies may land out of order); of the four, as many share the rows as there are blocks of 16 rows (one, two or four) and the rest
// splits the tile's positions.  Scores, maxima, sums and outputs are fp32; the weights are rounded to 16 bits for the second product, as the
// tensor cores take them.
#pragma once

#include "paged_work.cuh"

namespace b200ipc {

constexpr int kNarRows = 64;
constexpr int kNarTile = 64;     // positions
constexpr int kNarStages = 6;    // even: a stage belongs to one half of the warps
constexpr int kNarWarps = 8;     // that compute
constexpr int kNarThreads = (kNarWarps + 1) * 32;
constexpr int kNarTileBytes = kNarTile * kAttnD * 2;  // of K or V
constexpr int kNarORow = kAttnD + 4;                  // floats of a row of the merge buffer
constexpr size_t kNarSmem = 1024 + size_t(kNarStages) * 2 * kNarTileBytes + size_t(4) * 16 * kNarORow * 4;
constexpr int kNarStart = 1;     // what an item's start and end cost, in tiles
constexpr int kNarLeast = 2;     // a span is at least so long: more than kNarStart, so that every cut leaves a tile on both sides

struct NarrowCut {
  const PagedArgs& a;
  __device__ __forceinline__ bool takes(const Request& r) const { return r.n > 0 && r.n * a.group <= a.narrow_rows; }
  __device__ __forceinline__ int tiles(const Request& r) const { return (r.len + kNarTile - 1) / kNarTile; }
  __device__ __forceinline__ int64_t length(const Request& r) const { return takes(r) ? int64_t(a.hkv) * (kNarStart + tiles(r)) : 0; }
  __device__ __forceinline__ int4 place(const Mark& m) const {
    if (m.request >= a.requests) return make_int4(a.requests, 0, 0, 0);
    const int per = kNarStart + tiles(request_at(a, m.request));
    const int h = int(m.offset / per);
    return make_int4(m.request, h, max(0, int(m.offset - int64_t(h) * per) - kNarStart), 0);
  }
};

__device__ __forceinline__ void nar_ldmatrix(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void nar_ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void nar_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kNarWarps * 32) : "memory"); }

template <typename T>
__global__ void __launch_bounds__(kNarThreads, 1) paged_narrow_kernel(const __grid_constant__ PagedArgs args) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t full[kNarStages], empty[kNarStages];
  __shared__ Mark s_marks[2];
  __shared__ int s_abort;
  __shared__ float2 s_ml[4][16];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_o = reinterpret_cast<float*>(ring + kNarStages * 2 * kNarTileBytes);  // [4][16][kNarORow]
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = int(threadIdx.x & 31);
  volatile int* abort_flag = &s_abort;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kNarStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  const NarrowCut cut{args};
  find_span<kNarThreads>(args, [&](const Request& r) { return cut.length(r); }, kNarLeast, s_marks);
  const int4 first = cut.place(s_marks[0]), last = cut.place(s_marks[1]);
  if (threadIdx.x == 0) {
    args.starts[blockIdx.x] = first;
    if (blockIdx.x == gridDim.x - 1) args.starts[gridDim.x] = last;
  }
  lead<T>(args);
  const auto takes = [&](const Request& r) { return cut.takes(r); };
  Window win;

  // Every role walks the items of the span alike: f(request, its number, head, first tile, tile behind the last, tiles of the item).
  auto walk = [&](auto&& f) {
    int i = first.x < args.requests ? win.next(args, first.x, takes) : args.requests, h = first.y, t0 = first.z;
    while (i < args.requests && !(i > last.x || (i == last.x && (h > last.y || (h == last.y && t0 >= last.z))))) {
      const Request r = win.get(i);
      const int tiles = cut.tiles(r);
      f(r, i, h, t0, i == last.x && h == last.y ? last.z : tiles, tiles);
      t0 = 0;
      if (++h == args.hkv) {
        h = 0;
        i = win.next(args, i + 1, takes);
      }
    }
  };

  uint32_t st = 0, ph = 0;  // stage, and the parity of its round
  auto step = [&]() {
    if (++st == kNarStages) {
      st = 0;
      ph ^= 1u;
    }
  };
  if (warp == kNarWarps) {
    // ---- the stream: lane l loads box l / 4 of a tile, K or V, left or right half of the dimensions ----------------------
    const int box = min(args.page, kNarTile), boxes = kNarTile / box, per_page = args.page / box;
    const int sub = lane >> 2, half = lane & 1, value = (lane >> 1) & 1;
    const int64_t outside = args.pages * args.hkv * args.page;
    int issued = 0;
    walk([&](const Request& r, int i, int h, int t0, int t1, int) {
      const int* table = args.table + int64_t(i) * args.width;
      const int pages = (r.len + args.page - 1) / args.page;  // of the request
      int base = -64, entry = 0;                              // 32 entries of its table, one per lane
      for (int t = t0; t < t1; ++t) {
        // every lane's box: which page, and where in it
        const int b = t * boxes + sub, p = b / per_page, offset = (b - p * per_page) * box;
        const int p_first = t * boxes / per_page;
        if (p_first < base || (t * boxes + boxes - 1) / per_page >= base + 32) {
          base = p_first;
          entry = base + lane < pages ? table[base + lane] : -1;
        }
        const int64_t id = __shfl_sync(0xffffffffu, entry, min(31, p - base));
        const int n = min(boxes, (r.len - t * kNarTile + box - 1) / box);  // boxes that hold positions of the request
        mbar_wait_long(&empty[st], ph ^ 1u, abort_flag, kPagedTimeoutNs);
        if (__any_sync(0xffffffffu, *abort_flag)) return;
        if (lane == 0) mbar_expect_tx(&full[st], uint32_t(n * box) * kAttnD * 4u);
        __syncwarp();
        if (sub < n) {
          const int row = int(id >= 0 && id < args.pages ? (id * args.hkv + h) * args.page + offset : outside);
          unsigned char* dst = ring + st * 2 * kNarTileBytes + value * kNarTileBytes + half * (kNarTileBytes / 2) + sub * box * 128;
          tma_load_2d(dst, value ? &args.tma_v : &args.tma_k, &full[st], half * 64, row);
        }
        ++issued;
        step();
      }
    });
    // copies in flight land before the CTA leaves
    const uint64_t t0 = globaltimer_ns();
    for (int back = 1; back <= min(issued, kNarStages); ++back)
      mbar_drain(&full[(issued - back) % kNarStages], uint32_t((issued - back) / kNarStages) & 1u, t0);
  } else {
    // ---- the arithmetic ----------------------------------------------------------------------------------------------------
    const int side = warp >> 2, w4 = warp & 3, r8 = lane >> 2, c = lane & 3, G = args.group;
    const uint32_t ring_addr = smem_u32(ring);
    const uint32_t k_row = uint32_t(((lane >> 4) & 1) * 8 + (lane & 7)), k_chunk = (lane >> 3) & 1;
    const uint32_t v_row = uint32_t(((lane >> 3) & 1) * 8 + (lane & 7)), v_chunk = (lane >> 4) & 1;
    auto chunk_addr = [](uint32_t tile, uint32_t pos, uint32_t chunk) {
      return tile + (chunk >> 3) * (kNarTileBytes / 2) + pos * 128 + (((chunk & 7) ^ (pos & 7)) << 4);
    };
    walk([&](const Request& r, int, int h, int t0, int t1, int tiles) {
      const bool odd_tiles = t1 - t0 > 1 || (t1 - t0 == 1 && (st & 1u));  // whether warps 4-7 have any
      const int nrows = r.n * G, blocks = nrows <= 16 ? 1 : nrows <= 32 ? 2 : 4;
      const int block = w4 & (blocks - 1), slice = blocks == 1 ? w4 : blocks == 2 ? w4 >> 1 : 0;
      const int ra = block * 16 + r8, rb = ra + 8;  // this lane's two rows of the item
      const int ja = ra / G, jb = rb / G;
      auto row_of = [&](int row, int j) { return static_cast<const T*>(args.q) + int64_t(r.row0 + j) * args.row_stride + (int64_t(h) * G + (row - j * G)) * kAttnD; };
      uint32_t qa[8][4];
      {
        const uint32_t *pa = reinterpret_cast<const uint32_t*>(row_of(ra, ja)), *pb = reinterpret_cast<const uint32_t*>(row_of(rb, jb));
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          qa[k][0] = ra < nrows ? pa[8 * k + c] : 0u;
          qa[k][1] = rb < nrows ? pb[8 * k + c] : 0u;
          qa[k][2] = ra < nrows ? pa[8 * k + 4 + c] : 0u;
          qa[k][3] = rb < nrows ? pb[8 * k + 4 + c] : 0u;
        }
      }
      // positions that the rows see
      const int la = ra < nrows ? r.len - r.n + ja + 1 : 0, lb = rb < nrows ? r.len - r.n + jb + 1 : 0, all_see = r.len - r.n + 1;
      float ma = -INFINITY, mb = -INFINITY, sa = 0, sb = 0;
      float o[16][4];
#pragma unroll
      for (int t = 0; t < 16; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0;
      for (int t = t0; t < t1; ++t, step()) {
        if (int(st & 1u) != side) continue;
        if (!*abort_flag) mbar_wait_long(&full[st], ph, abort_flag, kPagedTimeoutNs);
        const uint32_t kt = ring_addr + st * 2 * kNarTileBytes, vt = kt + kNarTileBytes;
        for (int s16 = 0; s16 < blocks; ++s16) {
          const int at = slice * 16 * blocks + s16 * 16;  // first position within the tile
          const int pos = t * kNarTile + at;
          if (pos >= r.len) break;
          float s[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            uint32_t kf[4];
            nar_ldmatrix(kf, chunk_addr(kt, at + k_row, 2 * k + k_chunk));
            mma_16816<T>(s[0], qa[k][0], qa[k][1], qa[k][2], qa[k][3], kf[0], kf[1]);
            mma_16816<T>(s[1], qa[k][0], qa[k][1], qa[k][2], qa[k][3], kf[2], kf[3]);
          }
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][e] *= args.scale_log2;
          const bool masked = pos + 16 > all_see;
          if (masked) {
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
          if (pos + 16 > r.len) {
            const int left = r.len - pos - 2 * c;
            keep0 = left <= 0 ? 0u : left == 1 ? 0xffffu : 0xffffffffu;
            keep1 = left <= 8 ? 0u : left == 9 ? 0xffffu : 0xffffffffu;
          }
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            uint32_t vf[4];
            nar_ldmatrix_trans(vf, chunk_addr(vt, at + v_row, 2 * d + v_chunk));
            mma_16816<T>(o[2 * d], pw[0], pw[1], pw[2], pw[3], vf[0] & keep0, vf[1] & keep1);
            mma_16816<T>(o[2 * d + 1], pw[0], pw[1], pw[2], pw[3], vf[2] & keep0, vf[3] & keep1);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
      }
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        sa += __shfl_xor_sync(0xffffffffu, sa, d);
        sb += __shfl_xor_sync(0xffffffffu, sb, d);
      }
      // ---- the odd tiles' warps hand over to the even ones', these to all ---------------------------------------------
      float* mine = s_o + w4 * 16 * kNarORow;
      auto put = [&]() {
#pragma unroll
        for (int d = 0; d < 16; ++d) {
          *reinterpret_cast<float2*>(mine + r8 * kNarORow + 8 * d + 2 * c) = make_float2(o[d][0], o[d][1]);
          *reinterpret_cast<float2*>(mine + (r8 + 8) * kNarORow + 8 * d + 2 * c) = make_float2(o[d][2], o[d][3]);
        }
        if (c == 0) {
          s_ml[w4][r8] = make_float2(ma, sa);
          s_ml[w4][r8 + 8] = make_float2(mb, sb);
        }
      };
      if (odd_tiles) {
        if (side == 1) put();
        nar_sync();
        if (side == 0) {
          const float2 a = s_ml[w4][r8], b = s_ml[w4][r8 + 8];
          const float na = fmaxf(ma, a.x), nb = fmaxf(mb, b.x);
          const float ua = na == -INFINITY ? 0.f : na, ub = nb == -INFINITY ? 0.f : nb;
          const float fa = exp2_fast(ma - ua), fb = exp2_fast(mb - ub), ga = exp2_fast(a.x - ua), gb = exp2_fast(b.x - ub);
          ma = na;
          mb = nb;
          sa = sa * fa + a.y * ga;
          sb = sb * fb + b.y * gb;
#pragma unroll
          for (int d = 0; d < 16; ++d) {
            const float2 x = *reinterpret_cast<const float2*>(mine + r8 * kNarORow + 8 * d + 2 * c);
            const float2 y = *reinterpret_cast<const float2*>(mine + (r8 + 8) * kNarORow + 8 * d + 2 * c);
            o[d][0] = o[d][0] * fa + x.x * ga;
            o[d][1] = o[d][1] * fa + x.y * ga;
            o[d][2] = o[d][2] * fb + y.x * gb;
            o[d][3] = o[d][3] * fb + y.y * gb;
          }
        }
        __syncwarp();
      }
      if (side == 0) put();
      nar_sync();
      // 32 threads a row, four dimensions each
      const bool whole = t0 == 0 && t1 == tiles;
      float* piece = whole ? nullptr : Piece<kNarRows>::slot(args, blockIdx.x, t0 > 0 ? 0 : 1);
      const int slices = 4 / blocks;
      for (int row = warp; row < nrows; row += kNarWarps) {
        const int b = row >> 4, in = row & 15;
        float m = -INFINITY, l = 0;
        for (int s = 0; s < slices; ++s) m = fmaxf(m, s_ml[s * blocks + b][in].x);
        const float u = m == -INFINITY ? 0.f : m;
        float4 v = make_float4(0, 0, 0, 0);
        for (int s = 0; s < slices; ++s) {
          const float2 ml = s_ml[s * blocks + b][in];
          const float f = exp2_fast(ml.x - u);
          const float4 x = *reinterpret_cast<const float4*>(s_o + ((s * blocks + b) * 16 + in) * kNarORow + lane * 4);
          l += ml.y * f;
          v = make_float4(v.x + x.x * f, v.y + x.y * f, v.z + x.z * f, v.w + x.w * f);
        }
        if (whole) {
          const float inv = l == 0 ? 0.f : 1 / l;  // a row that sees nothing
          const int j = row / G;
          T* dst = static_cast<T*>(args.out) + (int64_t(r.row0 + j) * args.hq + int64_t(h) * G + (row - j * G)) * kAttnD + lane * 4;
          *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
        } else {
          if (lane == 0) *reinterpret_cast<float2*>(piece + 2 * row) = make_float2(m, l);
          *reinterpret_cast<float4*>(piece + 2 * kNarRows + row * kAttnD + lane * 4) = v;
        }
      }
      nar_sync();
    });
  }
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) *args.status = 1;
}

constexpr int kNarJoin = 8;  // warps of a row: one request alone leaves a piece on every SM
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_narrow_join_kernel(const __grid_constant__ PagedArgs args, int spans) {
  pdl_launch_dependents();
  pdl_wait();
  join_rows<T, kNarRows, kNarJoin>(args, spans, [&](const int4& item, int row) -> T* {
    const Request r = request_at(args, item.x);
    if (row >= r.n * args.group) return nullptr;
    const int j = row / args.group;
    return static_cast<T*>(args.out) + (int64_t(r.row0 + j) * args.hq + int64_t(item.y) * args.group + (row - j * args.group)) * kAttnD;
  });
}

}  // namespace b200ipc
