// What the kernels of the attention over a paged cache share: their arguments, how the work is cut, and the kernel that joins the pieces.
//
// An item is what one CTA can do by itself: the query rows of a (request, KV head) (narrow kernel), or a tile of them (wide kernel), over
// the positions they see, in tiles of positions.  All items follow one another on one axis, each as long as its tiles and a constant for
// its start and end; the axis is cut into equal spans, one per CTA (one per SM).  So nobody waits for a longest request, and a single long
// one uses the whole GPU.  Every CTA finds its span itself from the lengths on the GPU: one round of loads and a scan, and the same
// rounding everywhere.
//
// An item that a cut goes through leaves pieces: fp32 sums, maxima and unscaled outputs in the workspace.  A CTA has at most two, the end of an
// item that began in an earlier span (slot 0) and the beginning of one that goes on in the next (slot 1); the join walks them in order, so the result does not
// depend on timing.
#pragma once

#include "../common/check.h"
#include "../fused/gemm_local.cuh"
#include "decode_math.cuh"
#include "paged_ops.h"

namespace b200ipc {

constexpr uint64_t kPagedTimeoutNs = 2000000000;  // a wait inside a CTA takes microseconds

struct PagedArgs {
  alignas(64) CUtensorMap tma_k, tma_v;  // [pages * hkv * page, 128], boxes of 64 columns x min(page, 64) rows
  const void* q;
  void* out;
  const int *table, *lens, *cu_new;
  int4* starts;     // [CTAs + 1]: request, item of it, tile: where each span starts
  float* part;      // [CTAs][2][piece rows][2 + 128]: see Piece
  int* status;      // 0, or 1 when a wait gave up
  int64_t row_stride;
  int rows, requests, hq, hkv, group;
  int page, width;
  int64_t pages;
  int narrow_rows;  // items of up to so many rows belong to the narrow kernel, the others to the wide one
  int leads;        // the call's first kernel: resets the status, and writes the rows behind the last request
  float scale_log2;
};

// 2^x in one instruction: relative error 2^-22, results below 2^-126 are zero.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Request {
  int row0, n, len;  // first row of q, new tokens, tokens in the cache
};
__device__ __forceinline__ Request request_at(const PagedArgs& a, int i) {
  Request r;
  r.row0 = min(max(a.cu_new[i], 0), a.rows);
  r.n = min(max(a.cu_new[i + 1], r.row0), a.rows) - r.row0;
  r.len = min(max(a.lens[i], 0), a.width * a.page);
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

struct Mark {
  int request;
  int64_t offset;  // on the request's own part of the axis
};
// Start and end of this CTA's span; for all threads of the block (THREADS of them).  `length` of a request: its part of the axis, 0 for one
// that is not this kernel's.  No span is shorter than `least` but where the axis ends.
template <int THREADS, typename Length>
__device__ __forceinline__ void find_span(const PagedArgs& a, Length length, int64_t least, Mark* s_marks /* shared [2] */) {
  __shared__ int64_t s_sum[THREADS / 32];
  const int lane = int(threadIdx.x & 31), warp = int(threadIdx.x >> 5);
  const int each = (a.requests + THREADS - 1) / THREADS, i0 = min(a.requests, int(threadIdx.x) * each), i1 = min(a.requests, i0 + each);
  int64_t mine = 0;
  for (int i = i0; i < i1; ++i) mine += length(request_at(a, i));
  int64_t in = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) in += x;
  }
  if (lane == 31) s_sum[warp] = in;
  if (threadIdx.x < 2) s_marks[threadIdx.x] = {a.requests, 0};
  __syncthreads();
  int64_t before = in - mine, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
  }
  const int64_t spans = min(int64_t(gridDim.x), max(int64_t(1), total / least));
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int64_t c = int64_t(blockIdx.x) + k;
    const int64_t at = c >= spans ? total : total / spans * c + total % spans * c / spans;
    if (at >= before && at < before + mine) {
      int64_t o = at - before;
      for (int i = i0; i < i1; ++i) {
        const int64_t len = length(request_at(a, i));
        if (o < len) {
          s_marks[k] = {i, o};
          break;
        }
        o -= len;
      }
    }
  }
  __syncthreads();
}

// A piece: [rows] pairs (maximum in the log2 domain, sum), then [rows][128] of the output, not divided by the sum.
template <int ROWS>
struct Piece {
  static constexpr size_t kFloats = size_t(ROWS) * (2 + kAttnD);
  __device__ static float* slot(const PagedArgs& a, int cta, int which) { return a.part + (size_t(cta) * 2 + size_t(which)) * kFloats; }
};

// What the call's first kernel does: the status is good, rows behind the last request are zeros.
template <typename T>
__device__ __forceinline__ void lead(const PagedArgs& a) {
  if (!a.leads) return;
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
  const int tail = min(max(a.cu_new[a.requests], 0), a.rows), vectors = a.hq * kAttnD / 8;
  for (int64_t row = int64_t(tail) + blockIdx.x; row < a.rows; row += gridDim.x)
    for (int v = int(threadIdx.x); v < vectors; v += int(blockDim.x))
      reinterpret_cast<uint4*>(static_cast<T*>(a.out) + row * a.hq * kAttnD)[v] = make_uint4(0, 0, 0, 0);
}

// ---- the join ---------------------------------------------------------------------------------------------------------
// Where an item starts in span c and goes on in the next, its pieces are weighted with 2^(maximum - greatest maximum) and added in order.  A
// row is WARPS warps' work, each takes every WARPS-th piece; kJoinThreads / 32 / WARPS rows a CTA, span blockIdx.x.  `locate(item, row)`: the output row.
constexpr int kJoinThreads = 256;
template <typename T, int ROWS, int WARPS, typename Locate>
__device__ __forceinline__ void join_rows(const PagedArgs& a, int spans, Locate locate) {
  constexpr int kWarps = kJoinThreads / 32;
  __shared__ float s_m[kWarps], s_l[kWarps];
  __shared__ __align__(16) float4 s_o[kWarps][32];
  const int c = int(blockIdx.x);
  const int4 here = a.starts[c], next = a.starts[c + 1];
  if (next.z == 0 || (here.x == next.x && here.y == next.y && here.z > 0)) return;  // nothing starts here that goes on
  const int warp = int(threadIdx.x >> 5), lane = int(threadIdx.x & 31);
  const int row = int(blockIdx.y) * (kWarps / WARPS) + warp / WARPS;
  T* dst = locate(next, row);
  if (__syncthreads_count(dst != nullptr) == 0) return;
  int pieces = 1;  // and one in each of the following spans that start inside of the item
  for (int k0 = c + 1; k0 < spans; k0 += kJoinThreads) {
    const int k = k0 + int(threadIdx.x);
    const int4 from = k < spans ? a.starts[k] : make_int4(-1, 0, 0, 0);
    pieces += __syncthreads_count(from.x == next.x && from.y == next.y && from.z > 0);
  }
  float m = -INFINITY, l = 0;
  float4 o = make_float4(0, 0, 0, 0);
  if (dst != nullptr) {
#pragma unroll 4
    for (int n = warp % WARPS; n < pieces; n += WARPS) {
      const float* p = Piece<ROWS>::slot(a, c + n, n == 0 ? 1 : 0);
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(p + 2 * row));
      const float4 v = __ldcg(reinterpret_cast<const float4*>(p + 2 * ROWS + size_t(row) * kAttnD + lane * 4));
      const float mn = fmaxf(m, ml.x), u = mn == -INFINITY ? 0.f : mn;
      const float c0 = exp2_fast(m - u), c1 = exp2_fast(ml.x - u);
      m = mn;
      l = l * c0 + ml.y * c1;
      o = make_float4(o.x * c0 + v.x * c1, o.y * c0 + v.y * c1, o.z * c0 + v.z * c1, o.w * c0 + v.w * c1);
    }
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  s_o[warp][lane] = o;
  __syncthreads();
  if (warp % WARPS == 0 && dst != nullptr) {
    m = -INFINITY;
    for (int w = 0; w < WARPS; ++w) m = fmaxf(m, s_m[warp + w]);
    l = 0;
    o = make_float4(0, 0, 0, 0);
    for (int w = 0; w < WARPS; ++w) {
      const float x = s_m[warp + w] == -INFINITY ? 0.f : exp2_fast(s_m[warp + w] - m);
      const float4 v = s_o[warp + w][lane];
      l += s_l[warp + w] * x;
      o = make_float4(o.x + v.x * x, o.y + v.y * x, o.z + v.z * x, o.w + v.w * x);
    }
    const float inv = l == 0 ? 0.f : 1 / l;
    *reinterpret_cast<uint2*>(dst + lane * 4) = make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
  }
}

}  // namespace b200ipc
