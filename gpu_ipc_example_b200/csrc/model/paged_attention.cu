// Attention of a step's new tokens over a paged cache: the simple form, one CTA per token and KV head.
#include "../common/check.h"
#include "../common/pdl.h"
#include "decode_math.cuh"
#include "paged_ops.h"

namespace b200ipc {
namespace {

// One warp per query head of the group, one position after the other, running maximum and sum in fp32.
template <typename T>
__global__ void paged_attention_simple_kernel(const T* q, int64_t row_stride, const T* kcache, const T* vcache, const int* table, const int* lens,
                                              const int* cu_new, T* out, PagedAttentionShape s, float scale_log2) {
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x, h = blockIdx.y, lane = int(threadIdx.x & 31), group = s.hq / s.hkv;
  int i = 0;
  while (i < s.requests && cu_new[i + 1] <= t) ++i;
  for (int g = int(threadIdx.x >> 5); g < group; g += int(blockDim.x >> 5)) {
  T* dst = out + (int64_t(t) * s.hq + h * group + g) * kAttnD + lane * 4;
  float o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0;
  if (i < s.requests) {
    const int limit = min(lens[i] - (cu_new[i + 1] - cu_new[i]) + (t - cu_new[i]) + 1, s.width * s.page);
    const T* qp = q + int64_t(t) * row_stride + (int64_t(h) * group + g) * kAttnD + lane * 4;
    for (int p = 0; p < limit; ++p) {
      const int64_t page = table[int64_t(i) * s.width + p / s.page];
      if (page < 0 || page >= s.pages) continue;
      const int64_t at = ((page * s.hkv + h) * s.page + p % s.page) * kAttnD + lane * 4;
      float x = 0;
      for (int e = 0; e < 4; ++e) x += float(qp[e]) * float(kcache[at + e]);
      for (int k = 16; k > 0; k >>= 1) x += __shfl_xor_sync(0xffffffffu, x, k);
      x *= scale_log2;
      const float mn = fmaxf(m, x), c = exp2f(m - mn), w = exp2f(x - mn);
      l = l * c + w;
      m = mn;
      for (int e = 0; e < 4; ++e) o[e] = o[e] * c + w * float(vcache[at + e]);
    }
  }
  for (int e = 0; e < 4; ++e) dst[e] = T(l > 0 ? o[e] / l : 0.f);
  }
}

}  // namespace

size_t paged_attention_workspace_bytes(int, int, int) { return 256; }

void paged_attention(DType t, const void* q, int64_t row_stride, const void* kcache, const void* vcache, const int* table, const int* lens,
                     const int* cu_new, void* out, void*, const PagedAttentionShape& s, int, cudaStream_t stream) {
  const float scale_log2 = 1.4426950408889634f / sqrtf(float(kAttnD));
  const dim3 grid(unsigned(s.rows), unsigned(s.hkv)), block(unsigned(32 * min(8, s.hq / s.hkv)));
  if (t == DType::F16)
    paged_attention_simple_kernel<__half><<<grid, block, 0, stream>>>(static_cast<const __half*>(q), row_stride, static_cast<const __half*>(kcache), static_cast<const __half*>(vcache), table, lens, cu_new, static_cast<__half*>(out), s, scale_log2);
  else
    paged_attention_simple_kernel<__nv_bfloat16><<<grid, block, 0, stream>>>(static_cast<const __nv_bfloat16*>(q), row_stride, static_cast<const __nv_bfloat16*>(kcache), static_cast<const __nv_bfloat16*>(vcache), table, lens, cu_new, static_cast<__nv_bfloat16*>(out), s, scale_log2);
  B200_CUDA_CHECK(cudaGetLastError());
}

}  // namespace b200ipc
