// Block tables and slot maps of a paged cache, built on the GPU from the requests' lengths, and their inverse.
//
// Both are a prefix sum over the requests (pages needed or given back, new tokens) and a scatter behind it.  Some kilobytes in and
// out: the call is bound by latency (launch, one round of loads, the scan, one round of stores), so one kernel does it all.  Every CTA
// of one cluster makes the same scan of all requests in its shared memory and then takes a share of the pages and tokens, whose request
// it finds by bisection.  The lengths are written in place, so a CTA writes only when all have read (the cluster's barrier), which is
// also why it is one cluster and not a grid.  Extend and trim of 32 requests by a token 5.8 us, of 512 requests by up to 64 tokens 11.7
// (in a graph); a call by itself takes 8 (extend, four outputs) and 6.5 (trim) of host time.
#include <climits>

#include "../common/check.h"
#include "../common/pdl.h"
#include "paged_ops.h"

namespace b200ipc {
namespace {

constexpr int kTabThreads = 512;
// Rows from which on eight CTAs share extend's scatter.  Below, one CTA is ahead by the cluster's launch and barrier: 512 rows of 64 requests 3.2 us
// with one and 3.7 with eight, 1024 level (3.4, 3.3), 2048 5.4 and 4.0, 4032 7.7 and 3.9.
constexpr int64_t kTabWide = 1024;
// Entries of the table from which on they share trim's.  How many pages come back is known on the GPU alone, so it goes by how many can: a table of
// 64 x 512 that gives back a page a request pays 0.4 us for the cluster, and where 2048 come back extend and trim take 11.5 us instead of 49.
constexpr int64_t kTrimWide = 32768;

struct Scan {
  long long a, b;
};
__device__ __forceinline__ Scan operator+(Scan x, Scan y) { return {x.a + y.a, x.b + y.b}; }

// Exclusive prefix of `v` over the block's threads, and the block's sum.
__device__ Scan block_scan(Scan v, Scan* sum) {
  __shared__ Scan s_warp[kTabThreads / 32];
  const int lane = int(threadIdx.x & 31), warp = int(threadIdx.x >> 5);
  Scan in = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, in.a, o), b = __shfl_up_sync(0xffffffffu, in.b, o);
    if (lane >= o) in = in + Scan{a, b};
  }
  if (lane == 31) s_warp[warp] = in;
  __syncthreads();
  Scan before{0, 0}, all{0, 0};
#pragma unroll
  for (int w = 0; w < kTabThreads / 32; ++w) {
    if (w == warp) before = all;
    all = all + s_warp[w];
  }
  __syncthreads();
  *sum = all;
  return Scan{before.a + in.a - v.a, before.b + in.b - v.b};
}

// The last i with start[i] <= x, where start[0] = 0 and start[n] > x.
__device__ __forceinline__ int find(const int* start, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int pages_of(int n, int page) { return n / page + (n % page != 0); }

// s_page [requests + 1], s_row [requests + 1]: exclusive prefixes of the pages and the new tokens; s_len [requests]
__global__ void __launch_bounds__(kTabThreads) paged_extend_kernel(int* table, int* lens, const int* new_lens, const int* free_pages, int* n_free,
                                                                   int* cu_new, int64_t* slots, int* positions, int* status, int requests,
                                                                   int width, int capacity, int page, int rows) {
  extern __shared__ int s_mem[];
  int *s_page = s_mem, *s_row = s_page + requests + 1, *s_len = s_row + requests + 1;
  __shared__ int s_bad;
  pdl_launch_dependents();
  pdl_wait();
  if (threadIdx.x == 0) s_bad = 0;
  __syncthreads();
  const int have = *n_free;
  const long long room = (long long)(width) * page;
  Scan carry{0, 0};
  for (int base = 0; base < requests; base += kTabThreads) {
    const int i = base + int(threadIdx.x);
    Scan v{0, 0};
    if (i < requests) {
      const int len = lens[i], add = new_lens[i];
      int bad = 0;
      if (len < 0 || add < 0) bad = kPagedNegative;
      else if ((long long)(len) + add > min(room, (long long)(INT_MAX))) bad = kPagedTooLong;
      else v = {pages_of(len + add, page) - pages_of(len, page), add};
      if (bad) atomicOr(&s_bad, bad);
      s_len[i] = len;
    }
    Scan sum;
    const Scan at = carry + block_scan(v, &sum);
    if (i < requests) {  // what does not fit an int is refused below
      s_page[i] = int(at.a);
      s_row[i] = int(at.b);
    }
    carry = carry + sum;
  }
  if (threadIdx.x == 0) {
    s_page[requests] = int(carry.a);
    s_row[requests] = int(carry.b);
  }
  if (gridDim.x > 1) cluster_barrier();
  else __syncthreads();
  int bad = s_bad;
  if (have < 0 || have > capacity || carry.a > have) bad |= kPagedNoPages;
  if (carry.b > rows) bad |= kPagedTooMany;
  const int taken = bad ? 0 : int(carry.a), tokens = bad ? 0 : int(carry.b);
  const int first = int(blockIdx.x * kTabThreads + threadIdx.x), step = int(gridDim.x) * kTabThreads;
  if (first == 0) {
    *status = bad;
    cu_new[requests] = tokens;
    if (!bad) *n_free = have - taken;
  }
  for (int i = first; i < requests; i += step) {
    cu_new[i] = bad ? 0 : s_row[i];
    if (!bad) lens[i] = s_len[i] + s_row[i + 1] - s_row[i];
  }
  for (int k = first; k < taken; k += step) {
    const int i = find(s_page, requests, k);
    table[size_t(i) * size_t(width) + size_t(pages_of(s_len[i], page) + k - s_page[i])] = free_pages[have - 1 - k];
  }
  for (int t = first; t < rows; t += step) {
    int64_t slot = -1;
    int pos = 0;
    if (t < tokens) {
      const int i = find(s_row, requests, t), old = pages_of(s_len[i], page);
      pos = s_len[i] + t - s_row[i];
      const int col = pos / page;
      const int at = col < old ? table[size_t(i) * size_t(width) + size_t(col)] : free_pages[have - 1 - (s_page[i] + col - old)];
      if (at >= 0) slot = int64_t(at) * page + (pos - col * page);
    }
    slots[t] = slot;
    positions[t] = pos;
  }
}

// s_page as above, s_keep [requests]: the lengths that stay
__global__ void __launch_bounds__(kTabThreads) paged_trim_kernel(int* table, int* lens, const int* keep_lens, int* free_pages, int* n_free,
                                                                 int* status, int requests, int width, int capacity, int page) {
  extern __shared__ int s_mem[];
  int *s_page = s_mem, *s_keep = s_page + requests + 1;
  __shared__ int s_bad;
  pdl_launch_dependents();
  pdl_wait();
  if (threadIdx.x == 0) s_bad = 0;
  __syncthreads();
  const int have = *n_free;
  const long long room = (long long)(width) * page;
  Scan carry{0, 0};
  for (int base = 0; base < requests; base += kTabThreads) {
    const int i = base + int(threadIdx.x);
    Scan v{0, 0};
    if (i < requests) {
      const int len = lens[i], keep = keep_lens[i];
      int bad = 0;
      if (len < 0 || keep < 0) bad = kPagedNegative;
      else if (keep > len || len > room) bad = kPagedTooLong;
      else v.a = pages_of(len, page) - pages_of(keep, page);
      if (bad) atomicOr(&s_bad, bad);
      s_keep[i] = keep;
    }
    Scan sum;
    const Scan at = carry + block_scan(v, &sum);
    if (i < requests) s_page[i] = int(at.a);
    carry = carry + sum;
  }
  if (threadIdx.x == 0) s_page[requests] = int(carry.a);
  if (gridDim.x > 1) cluster_barrier();
  else __syncthreads();
  int bad = s_bad;
  if (have < 0 || carry.a > (long long)(capacity) - have) bad |= kPagedNoPages;
  const int back = bad ? 0 : int(carry.a);
  const int first = int(blockIdx.x * kTabThreads + threadIdx.x), step = int(gridDim.x) * kTabThreads;
  if (first == 0) {
    *status = bad;
    if (!bad) *n_free = have + back;
  }
  if (!bad)
    for (int i = first; i < requests; i += step) lens[i] = s_keep[i];
  for (int k = first; k < back; k += step) {
    const int i = find(s_page, requests, k);
    int* entry = table + size_t(i) * size_t(width) + size_t(pages_of(s_keep[i], page) + k - s_page[i]);
    free_pages[have + back - 1 - k] = *entry;  // the order that paged_extend took them in, backwards
    *entry = -1;
  }
}

constexpr size_t extend_smem(int requests) { return size_t(3 * requests + 2) * sizeof(int); }
constexpr size_t trim_smem(int requests) { return size_t(2 * requests + 1) * sizeof(int); }

// `most`: of a call with as many requests as there can be.  The limit is always set to that, as another thread may be about to launch.
template <typename... Params, typename... Args>
void launch_one_cluster(void (*kernel)(Params...), int ctas, size_t smem, size_t most, cudaStream_t stream, Args... args) {
  if (smem > 48 * 1024) B200_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(most)));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(kTabThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (ctas > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = unsigned(ctas);
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  B200_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...));
}

}  // namespace

void paged_extend(int* table, int* lens, const int* new_lens, const int* free_pages, int* n_free, int* cu_new, int64_t* slots, int* positions,
                  int* status, int requests, int width, int capacity, int page, int rows, cudaStream_t stream) {
  B200_REQUIRE(requests >= 1 && requests <= kPagedMaxRequests && width >= 1 && page >= 1 && rows >= 0 && capacity >= 0, "paged_extend: bad sizes");
  launch_one_cluster(paged_extend_kernel, rows >= kTabWide ? 8 : 1, extend_smem(requests), extend_smem(kPagedMaxRequests), stream, table, lens, new_lens,
                     free_pages, n_free, cu_new, slots, positions, status, requests, width, capacity, page, rows);
}

void paged_trim(int* table, int* lens, const int* keep_lens, int* free_pages, int* n_free, int* status, int requests, int width, int capacity,
                int page, cudaStream_t stream) {
  B200_REQUIRE(requests >= 1 && requests <= kPagedMaxRequests && width >= 1 && page >= 1 && capacity >= 0, "paged_trim: bad sizes");
  launch_one_cluster(paged_trim_kernel, int64_t(requests) * width >= kTrimWide ? 8 : 1, trim_smem(requests), trim_smem(kPagedMaxRequests), stream, table,
                     lens, keep_lens, free_pages, n_free, status, requests, width, capacity, page);
}

}  // namespace b200ipc
