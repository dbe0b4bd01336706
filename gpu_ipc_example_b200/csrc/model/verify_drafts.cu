// Verification of drafted tokens against the target's probabilities (speculative sampling, Leviathan et al. 2023), from random numbers
// that the caller gives:
//
//   draft j of a request is accepted while  accept[j] * q_j(d_j) < p_j(d_j)
//   behind n accepted ones comes one more word: with weights max(p_n - q_n, 0) where draft n was turned down (p_n where these are all
//   zero), p_n where there is no draft n; it is the first word whose running sum is above sample * (sum of the weights).
//
// Products, differences and sums are taken in 64 bits: a product of two fp32 numbers is exact there, and a running sum over a vocabulary
// is good to 1e-13, so that the words do not depend on the order of the additions (in 32 bits one draw in a hundred would).  With NaN every
// comparison fails: a word of NaN has no weight in p, nor in max(p - q, 0) where either is NaN, and a draft whose p or q is NaN is turned down.
//
// Bound by memory: of all the rows one of p and one of q is read, 8 bytes a word.  A request is a cluster of CTAs, each with a piece of
// the vocabulary, each of its warps with a run of it; the sums of all warps are exchanged through distributed shared memory, every CTA
// adds them in the same order, and the one warp whose run holds the sampled place reads that run again (from L1 or L2).  32 requests,
// four drafts, 128256 words: 10.9 us (10.2 without the drafts' probabilities; of 32000 words 7.4 and 7.1), of which 21.6 MB of memory traffic are
// 3.3; the rest is a chain of launch, gathers of the drafts' words, the stream's first arrival, the exchange and the second reading.  With
// loads that the compiler issued one round at a time it was 15.
#include "../common/check.h"
#include "../common/pdl.h"
#include "paged_ops.h"

namespace b200ipc {
namespace {

constexpr int kVerThreads = 512;
constexpr int kVerWarps = kVerThreads / 32;
constexpr int kVerCluster = 8;
constexpr int kVerRuns = kVerWarps * kVerCluster;

struct VerifyArgs {
  const float *target, *draft;  // draft nullptr: the draft is certain of its token
  const int64_t* tokens;
  const int* draft_lens;        // nullptr: all of them
  const float *accept, *sample;
  int64_t* out;
  int* accepted;
  VerifyShape s;
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// The weights of a row.  q nullptr: p alone; else max(p - q, 0).  spare: a word without weight, or -1.
struct Weights {
  const float *p, *q;
  int64_t spare;
  __device__ __forceinline__ double of(float x, float y, int64_t i) const {
    const double d = double(x) - double(y);
    return d > 0 && i != spare ? d : 0.0;
  }
  __device__ __forceinline__ double of4(const float4& x, const float4& y, int64_t i) const {
    return (of(x.x, y.x, i) + of(x.y, y.y, i + 1)) + (of(x.z, y.z, i + 2) + of(x.w, y.w, i + 3));
  }
  __device__ __forceinline__ double at(int64_t i) const { return of(p[i], q ? q[i] : 0.f, i); }
};

__device__ __forceinline__ double warp_sum(double s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
__device__ __forceinline__ double warp_prefix(double s, int lane) {  // of this lane's value and those before
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double x = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += x;
  }
  return s;
}
// Sum of the words [i0, i1) by one warp; the same order in every call.
__device__ double run_sum(const Weights& w, int64_t i0, int64_t i1, int lane, bool vec) {
  double s = 0;
  if (vec) {  // four vectors of each row on their way at a time
    for (int64_t b = i0 + lane * 4; b < i1; b += 512) {
      float4 x[4], y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t i = b + k * 128;
        x[k] = i < i1 ? *reinterpret_cast<const float4*>(w.p + i) : make_float4(0, 0, 0, 0);
        y[k] = i < i1 && w.q ? *reinterpret_cast<const float4*>(w.q + i) : make_float4(0, 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) s += w.of4(x[k], y[k], b + k * 128);
    }
  } else {
#pragma unroll 8
    for (int64_t i = i0 + lane; i < i1; i += 32) s += w.at(i);
  }
  return warp_sum(s);
}
struct Found {
  int at;         // the first place with a value whose running sum is above `goal`, else the last one with a value; -1: there is none
  double before;  // the sum in front of it
};
// Among `value`s of the lanes, behind a sum of `start`.
__device__ __forceinline__ Found find(double value, double start, double goal, int lane) {
  const double in = warp_prefix(value, lane);
  const unsigned some = __ballot_sync(0xffffffffu, value > 0), over = __ballot_sync(0xffffffffu, value > 0 && start + in > goal);
  if (some == 0) return {-1, start};
  const int at = over ? __ffs(int(over)) - 1 : 31 - __clz(int(some));
  const double before = __shfl_sync(0xffffffffu, in - value, at);
  return {at, start + before};
}

__global__ void __launch_bounds__(kVerThreads) verify_drafts_kernel(const VerifyArgs a) {
  __shared__ double s_runs[2][kVerRuns];
  pdl_launch_dependents();
  cluster_arrive();
  pdl_wait();
  const int64_t r = blockIdx.x / kVerCluster;
  const int part = int(blockIdx.x % kVerCluster), warp = int(threadIdx.x >> 5), lane = int(threadIdx.x & 31);
  const int K = a.s.drafts;
  const int64_t V = a.s.vocab;
  const int64_t* tokens = a.tokens + r * K;
  const float* target = a.target + r * a.s.target_b;
  const float* draft = a.draft ? a.draft + r * a.s.draft_b : nullptr;
  const int len = a.draft_lens ? max(0, min(K, a.draft_lens[r])) : K;
  // every warp looks at the drafts itself, 32 of them a time
  int n = len;
  for (int j0 = 0; j0 < len && n == len; j0 += 32) {
    const int j = j0 + lane;
    bool good = true;
    if (j < len) {
      const int64_t d = tokens[j];
      good = false;
      if (d >= 0 && d < V) {
        const double q = draft ? double(draft[j * a.s.draft_j + d]) : 1.0;
        good = double(a.accept[r * K + j]) * q < double(target[j * a.s.target_j + d]);
      }
    }
    const unsigned no = __ballot_sync(0xffffffffu, !good);
    if (no) n = j0 + __ffs(int(no)) - 1;
  }
  const bool turned_down = n < len;
  Weights w{target + n * a.s.target_j, turned_down && draft ? draft + n * a.s.draft_j : nullptr, turned_down && !draft ? tokens[n] : -1};
  const int64_t per = ((V + kVerRuns - 1) / kVerRuns + 127) / 128 * 128;  // words of a warp's run
  const int run = part * kVerWarps + warp;
  const int64_t i0 = min(V, run * per), i1 = min(V, i0 + per);
  // vectors of four, where every row starts on one
  auto vectors = [&](const Weights& x) {
    return V % 4 == 0 && (reinterpret_cast<uintptr_t>(x.p) & 15) == 0 && (reinterpret_cast<uintptr_t>(x.q) & 15) == 0;
  };
  auto exchange = [&](double mine, double* runs) {  // every CTA of the cluster gets every run's sum
    if (lane < kVerCluster) {
      uint32_t to;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(uint32_t(__cvta_generic_to_shared(runs + run))), "r"(lane));
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(mine) : "memory");
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    double sum = 0;
#pragma unroll
    for (int i = 0; i < kVerRuns / 32; ++i) sum += runs[lane * (kVerRuns / 32) + i];
    return warp_sum(sum);
  };
  const double* runs = s_runs[0];
  const double first = run_sum(w, i0, i1, lane, vectors(w));
  __syncwarp();
  cluster_wait();  // the others have started: their shared memory can be written
  double total = exchange(first, s_runs[0]);
  if (turned_down && !(total > 0)) {  // the target gives no word more than the draft does: its own probabilities
    w.q = nullptr;
    w.spare = -1;
    total = exchange(run_sum(w, i0, i1, lane, vectors(w)), s_runs[1]);
    runs = s_runs[1];
  }
  const double goal = double(a.sample[r]) * total;
  // The run, then the lane's stretch of it, then the word.  Where no running sum is above the goal (rounding, or a number that is not below
  // one) it is the last with a weight.
  constexpr int kEach = kVerRuns / 32;
  double sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) sum += runs[lane * kEach + i];
  const Found lanes = find(sum, 0, goal, lane);
  int chosen = -1;
  double before = lanes.before;
  if (lanes.at >= 0) {
    const Found f = find(lane < kEach ? runs[lanes.at * kEach + lane] : 0, before, goal, lane);
    chosen = lanes.at * kEach + f.at;
    before = f.before;
  }
  int64_t word = -1;
  if (chosen >= 0 ? run == chosen : run == 0) {
    if (chosen >= 0) {
      const int64_t stretch = per / 32;
      double mine = 0;
      const int64_t s0 = i0 + lane * stretch, s1 = min(i1, s0 + stretch);
      if (vectors(w)) {  // a stretch is whole vectors
#pragma unroll 8
        for (int64_t i = s0; i < s1; i += 4)
          mine += w.of4(*reinterpret_cast<const float4*>(w.p + i), w.q ? *reinterpret_cast<const float4*>(w.q + i) : make_float4(0, 0, 0, 0), i);
      } else {
#pragma unroll 8
        for (int64_t i = s0; i < s1; ++i) mine += w.at(i);
      }
      const Found f = find(mine, before, goal, lane);
      double at = f.before;
      int64_t some = -1;
      for (int64_t k = 0; k < stretch && word < 0; k += 32) {
        const int64_t i = i0 + f.at * stretch + k + lane;
        const double x = k + lane < stretch && i < i1 ? w.at(i) : 0.0;
        const double in = warp_prefix(x, lane);
        const unsigned over = __ballot_sync(0xffffffffu, x > 0 && at + in > goal), any = __ballot_sync(0xffffffffu, x > 0);
        if (over) word = i - lane + __ffs(int(over)) - 1;
        if (any) some = i - lane + 31 - __clz(int(any));
        at += __shfl_sync(0xffffffffu, in, 31);
      }
      if (word < 0) word = some;
    }
    for (int j = lane; j <= K; j += 32) a.out[r * (K + 1) + j] = j < n ? tokens[j] : j == n ? word : -1;
    if (lane == 0) a.accepted[r] = n;
  }
}

}  // namespace

void verify_drafts(const float* target, const float* draft, const int64_t* tokens, const int* draft_lens, const float* accept, const float* sample,
                   int64_t* out, int* accepted, const VerifyShape& s, cudaStream_t stream) {
  B200_REQUIRE(s.requests >= 0 && s.drafts >= 0 && s.vocab >= 1, "verify_drafts: bad sizes");
  if (s.requests == 0) return;
  const VerifyArgs a{target, draft, tokens, draft_lens, accept, sample, out, accepted, s};
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(s.requests) * kVerCluster);
  cfg.blockDim = dim3(kVerThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kVerCluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2u : 1u;
  B200_CUDA_CHECK(cudaLaunchKernelEx(&cfg, verify_drafts_kernel, a));
}

}  // namespace b200ipc
