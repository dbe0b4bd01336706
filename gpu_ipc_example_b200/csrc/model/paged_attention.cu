// Attention of a step's new tokens over a paged cache: which kernels a call takes.
#include "paged_narrow.cuh"

#include "../common/cu_driver.h"

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

// K or V as rows of 128, in boxes of half a row (a swizzle row) by what a page and a tile have in common.  Made anew for each call.
CUtensorMap cache_map(DType t, const void* cache, const PagedAttentionShape& s) {
  CUtensorMap map;
  cuuint64_t dims[2] = {cuuint64_t(kAttnD), cuuint64_t(s.pages) * cuuint64_t(s.hkv) * cuuint64_t(s.page)};
  cuuint64_t strides[1] = {kAttnD * 2};
  cuuint32_t box[2] = {64, cuuint32_t(std::min(s.page, kNarTile))}, one[2] = {1, 1};
  B200_CU_CHECK(cu().TensorMapEncodeTiled(&map, t == DType::F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                                          const_cast<void*>(cache), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE));
  return map;
}

// The workspace: a status word, then for each kernel where the spans start, then the pieces.
constexpr size_t kHead = 256;
size_t round_up(size_t n) { return (n + 255) / 256 * 256; }
size_t starts_bytes(int spans) { return round_up(size_t(spans + 1) * sizeof(int4)); }
template <int ROWS>
size_t pieces_bytes(int spans) { return round_up(size_t(spans) * 2 * Piece<ROWS>::kFloats * sizeof(float)); }

template <typename T>
void launch_narrow(PagedArgs& a, int spans, char* workspace, int most_rows, cudaStream_t stream) {
  a.starts = reinterpret_cast<int4*>(workspace);
  a.part = reinterpret_cast<float*>(workspace + starts_bytes(spans));
  const void* kernel = reinterpret_cast<const void*>(&paged_narrow_kernel<T>);
  B200_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kNarSmem)));
  void* params[] = {&a};
  B200_CUDA_CHECK(launch_maybe_pdl(kernel, dim3(unsigned(spans)), dim3(kNarThreads), params, kNarSmem, stream, true));
  void* join[] = {&a, &spans};
  B200_CUDA_CHECK(launch_maybe_pdl(reinterpret_cast<const void*>(&paged_narrow_join_kernel<T>), dim3(unsigned(spans), unsigned(most_rows)), dim3(kJoinThreads), join, 0,
                                   stream, true));
}

}  // namespace

size_t paged_attention_workspace_bytes(int group, int max_new, int sm_count) {
  return kHead + starts_bytes(sm_count) + pieces_bytes<kNarRows>(sm_count);
}

void paged_attention(DType t, const void* q, int64_t row_stride, const void* kcache, const void* vcache, const int* table, const int* lens,
                     const int* cu_new, void* out, void* workspace, const PagedAttentionShape& s, int sm_count, cudaStream_t stream) {
  PagedArgs a{};
  a.tma_k = cache_map(t, kcache, s);
  a.tma_v = cache_map(t, vcache, s);
  a.q = q;
  a.out = out;
  a.table = table;
  a.lens = lens;
  a.cu_new = cu_new;
  a.status = static_cast<int*>(workspace);
  a.row_stride = row_stride;
  a.rows = s.rows;
  a.requests = s.requests;
  a.hq = s.hq;
  a.hkv = s.hkv;
  a.group = s.hq / s.hkv;
  a.page = s.page;
  a.width = s.width;
  a.pages = s.pages;
  a.narrow_rows = kNarRows;
  a.leads = 1;
  a.scale_log2 = 1.4426950408889634f / sqrtf(float(kAttnD));
  const int64_t most = int64_t(s.max_new) * a.group;
  char* ws = static_cast<char*>(workspace) + kHead;
  if (most > kNarRows) {
    const dim3 grid(unsigned(s.rows), unsigned(s.hkv)), block(unsigned(32 * min(8, s.hq / s.hkv)));
    if (t == DType::F16)
      paged_attention_simple_kernel<__half><<<grid, block, 0, stream>>>(static_cast<const __half*>(q), row_stride, static_cast<const __half*>(kcache), static_cast<const __half*>(vcache), table, lens, cu_new, static_cast<__half*>(out), s, a.scale_log2);
    else
      paged_attention_simple_kernel<__nv_bfloat16><<<grid, block, 0, stream>>>(static_cast<const __nv_bfloat16*>(q), row_stride, static_cast<const __nv_bfloat16*>(kcache), static_cast<const __nv_bfloat16*>(vcache), table, lens, cu_new, static_cast<__nv_bfloat16*>(out), s, a.scale_log2);
    B200_CUDA_CHECK(cudaGetLastError());
    return;
  }
  (t == DType::F16 ? launch_narrow<__half> : launch_narrow<__nv_bfloat16>)(a, sm_count, ws, int(std::min<int64_t>(most, kNarRows)), stream);
}

}  // namespace b200ipc
