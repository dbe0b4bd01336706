// Attention of a step's new tokens over a paged cache: which kernels a call takes.
#include "paged_narrow.cuh"
#include "paged_wide.cuh"

#include <atomic>

#include "../common/cu_driver.h"

namespace b200ipc {
namespace {

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

// Q so that 128 rows of an item, heads of a group side by side, are one box for each half of the dimensions.
CUtensorMap query_map(DType t, const PagedArgs& a) {
  CUtensorMap map;
  const cuuint64_t head = kAttnD * 2, stride = a.rows > 1 ? cuuint64_t(a.row_stride) * 2 : cuuint64_t(a.hq) * head;
  cuuint64_t dims[5] = {64, 2, cuuint64_t(a.group), cuuint64_t(a.hkv), cuuint64_t(a.rows)};
  cuuint64_t strides[4] = {128, head, head * cuuint64_t(a.group), stride};
  cuuint32_t box[5] = {64, 1, cuuint32_t(a.group), 1, cuuint32_t(128 / a.group)}, one[5] = {1, 1, 1, 1, 1};
  B200_CU_CHECK(cu().TensorMapEncodeTiled(&map, t == DType::F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
                                          const_cast<void*>(a.q), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE));
  return map;
}

// The workspace: a status word; the narrow kernel's counters, zero between calls; its pieces, or where the wide kernel's spans start and its pieces.
constexpr size_t kHead = 256;
size_t round_up(size_t n) { return (n + 255) / 256 * 256; }
size_t starts_bytes(int spans) { return round_up(size_t(spans + 1) * sizeof(Start)); }
size_t counters_bytes(int spans) { return round_up(size_t(spans) * sizeof(unsigned int)); }
template <int ROWS>
size_t pieces_bytes(int spans) { return round_up(size_t(spans) * 2 * Piece<ROWS>::kFloats * sizeof(float)); }

// The limit on a kernel's shared memory, set once per kernel and GPU.
template <typename T, int ROWS>
void allow_smem(const void* kernel, size_t smem) {
  static std::atomic<uint64_t> done{0};
  int device = 0;
  B200_CUDA_CHECK(cudaGetDevice(&device));
  const uint64_t bit = uint64_t(1) << (device & 63);
  if (device < 64 && (done.load(std::memory_order_relaxed) & bit)) return;
  B200_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
  done.fetch_or(bit, std::memory_order_relaxed);
}

template <typename T>
void run(PagedArgs& a, const PagedAttentionShape& s, char* workspace, int spans, cudaStream_t stream) {
  void* params[] = {&a, &spans};
  // Up to 16 rows for every request: the narrow kernel.  A batch with longer ones is the wide kernel's as a whole, which for single tokens alone is
  // behind by 7 us a call (32 x 2048 15.5 and 22.8 us, 16 x 32768 53.1 and 59.6), but has them read while it computes for
  // the others (a chunk of 2047 tokens among 23 requests 170 us with both kernels, 147 with this one).
  const int64_t most = int64_t(s.max_new) * a.group;
  if (most <= kNarRows) {
    const void* kernel = reinterpret_cast<const void*>(&paged_narrow_kernel<T>);
    a.arrived = reinterpret_cast<unsigned int*>(workspace);
    a.part = reinterpret_cast<float*>(workspace + counters_bytes(spans));
    allow_smem<T, kNarRows>(kernel, kNarSmem);
    B200_CUDA_CHECK(launch_maybe_pdl(kernel, dim3(unsigned(spans)), dim3(kNarThreads), params, kNarSmem, stream, true));
    return;
  }
  const void* kernel = reinterpret_cast<const void*>(&paged_wide_kernel<T>);
  workspace += counters_bytes(spans);  // which stay zero
  a.starts = reinterpret_cast<Start*>(workspace);
  a.part = reinterpret_cast<float*>(workspace + starts_bytes(spans));
  a.q_boxes = 128 % a.group == 0;
  if (a.q_boxes) a.tma_q = query_map(std::is_same<T, __half>::value ? DType::F16 : DType::BF16, a);
  allow_smem<T, kWideRows>(kernel, kWideSmem);
  B200_CUDA_CHECK(launch_maybe_pdl(kernel, dim3(unsigned(spans)), dim3(kWideThreads), params, kWideSmem, stream, true));
  const unsigned groups = unsigned((std::min<int64_t>(most, kWideRows) + kJoinRows - 1) / kJoinRows);
  B200_CUDA_CHECK(launch_maybe_pdl(reinterpret_cast<const void*>(&paged_join_kernel<T, kWideRows>), dim3(unsigned(spans), groups), dim3(kJoinThreads), params, 0, stream,
                                   true));
}

}  // namespace

size_t paged_attention_workspace_bytes(int group, int max_new, int sm_count) {
  const bool wide = int64_t(max_new) * group > kNarRows;
  return kHead + counters_bytes(sm_count) + (wide ? starts_bytes(sm_count) + pieces_bytes<kWideRows>(sm_count) : pieces_bytes<kNarRows>(sm_count));
}

void paged_attention(DType t, const void* q, int64_t row_stride, const void* kcache, const void* vcache, const int* table, const int* lens,
                     const int* cu_new, void* out, void* workspace, const PagedAttentionShape& s, int sm_count, uint64_t timeout_ns, uint32_t flags,
                     cudaStream_t stream) {
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
  a.max_new = s.max_new;
  while ((1 << a.page_log) < s.page) ++a.page_log;
  a.width = s.width;
  a.pages = s.pages;
  a.scale_log2 = 1.4426950408889634f / sqrtf(float(kAttnD));
  a.timeout_ns = timeout_ns;
  a.mute = (flags & kMuteSends) != 0;
  (t == DType::F16 ? run<__half> : run<__nv_bfloat16>)(a, s, static_cast<char*>(workspace) + kHead, sm_count, stream);
}

}  // namespace b200ipc
