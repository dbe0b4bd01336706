// Rotary positions of a step's new tokens and the append of their keys and values to a paged cache, in one pass.
//
// (x_i, x_{i+64}) of every query and key head turns by the angle position * theta^(-i/64).  Positions go far (100000 and more), and an
// angle in 32 bits is then off by 1e-2 of a radian, so the angle and its reduction to one turn are computed in 64 bits, once per
// token and pair for all heads; the reduced angle, its sine and cosine and the rotation are in 32 bits, with one rounding at the end.
//
// Bound by memory: (hq + 2 hkv) x 256 bytes in and out per token.  One CTA per token: 16-byte loads and stores, eight pairs a thread
// (two vectors 64 elements apart), the loads of a thread's first heads in flight while the angles are computed.  4001 tokens of
// 64 + 2 x 8 heads, 167 MB in and out: 28.5 us, 5.9 TB/s; 32 tokens: 1.9 us in a graph.
#include "../common/check.h"
#include "../common/pdl.h"
#include "decode_math.cuh"
#include "paged_ops.h"

namespace b200ipc {
namespace {

constexpr int kAppThreads = 128;

struct Frequencies {
  double inv[kAttnD / 2];  // theta^(-i / 64)
};

template <typename T>
__global__ void __launch_bounds__(kAppThreads) rope_paged_append_kernel(const T* qkv, int64_t row_stride, T* q_out, T* kcache, T* vcache,
                                                                        const int64_t* slots, const int* positions, int hq, int hkv, int page,
                                                                        int64_t pages, const __grid_constant__ Frequencies freq) {
  using T2 = typename Num<T>::T2;
  pdl_launch_dependents();
  pdl_wait();
  constexpr int half = kAttnD / 2, kItems = half / 8;  // vectors of half a head
  __shared__ __align__(16) float s_sin[half], s_cos[half];
  const int64_t t = blockIdx.x;
  const T* row = qkv + t * row_stride;
  const int64_t slot = slots[t];
  const bool live = slot >= 0 && slot < pages * page;
  // a thread takes the same vector (eight pairs) of every kAppThreads / kItems-th head
  const int e = int(threadIdx.x % kItems) * 8, first = int(threadIdx.x / kItems);
  constexpr int kStep = kAppThreads / kItems;
  const int heads = live ? hq + 2 * hkv : hq;
  uint4 a{}, b{};
  if (first < heads) {
    a = *reinterpret_cast<const uint4*>(row + int64_t(first) * kAttnD + e);
    b = *reinterpret_cast<const uint4*>(row + int64_t(first) * kAttnD + e + half);
  }
  if (threadIdx.x < half) {
    constexpr double kTurn = 6.283185307179586476925;
    const double angle = double(positions[t]) * freq.inv[threadIdx.x];
    const float r = float(fma(-rint(angle * (1.0 / kTurn)), kTurn, angle));
    float sn, cs;
    sincosf(r, &sn, &cs);
    s_sin[threadIdx.x] = sn;
    s_cos[threadIdx.x] = cs;
  }
  __syncthreads();
  float sn[8], cs[8];
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    *reinterpret_cast<float4*>(sn + i) = *reinterpret_cast<const float4*>(s_sin + e + i);
    *reinterpret_cast<float4*>(cs + i) = *reinterpret_cast<const float4*>(s_cos + e + i);
  }
  const int64_t at_page = live ? slot / page : 0, at = live ? slot - at_page * page : 0;
  for (int h = first; h < heads;) {
    uint4 na{}, nb{};
    const int next = h + kStep;
    if (next < heads) {
      na = *reinterpret_cast<const uint4*>(row + int64_t(next) * kAttnD + e);
      nb = *reinterpret_cast<const uint4*>(row + int64_t(next) * kAttnD + e + half);
    }
    T* dst;
    if (h < hq) {
      dst = q_out + (t * hq + h) * kAttnD;
    } else {
      const bool key = h < hq + hkv;
      dst = (key ? kcache : vcache) + ((at_page * hkv + (key ? h - hq : h - hq - hkv)) * page + at) * kAttnD;
    }
    if (h < hq + hkv) {
      T2 *pa = reinterpret_cast<T2*>(&a), *pb = reinterpret_cast<T2*>(&b);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = Num<T>::up(pa[i]), y = Num<T>::up(pb[i]);
        const float2 u = rope_pair(x.x, y.x, sn[2 * i], cs[2 * i]), v = rope_pair(x.y, y.y, sn[2 * i + 1], cs[2 * i + 1]);
        pa[i] = Num<T>::down(u.x, v.x);
        pb[i] = Num<T>::down(u.y, v.y);
      }
    }
    *reinterpret_cast<uint4*>(dst + e) = a;
    *reinterpret_cast<uint4*>(dst + e + half) = b;
    a = na;
    b = nb;
    h = next;
  }
}

}  // namespace

void rope_paged_append(DType t, const void* qkv, int64_t row_stride, void* q_out, void* kcache, void* vcache, const int64_t* slots,
                       const int* positions, int rows, int hq, int hkv, int page, int64_t pages, double theta, cudaStream_t stream) {
  B200_REQUIRE(rows >= 0 && hq >= 1 && hkv >= 1 && page >= 1 && pages >= 0 && theta > 0, "rope_paged_append: bad sizes");
  if (rows == 0) return;
  static thread_local double made_for = 0;  // 64 powers are a microsecond
  static thread_local Frequencies f;
  if (made_for != theta) {
    for (int i = 0; i < kAttnD / 2; ++i) f.inv[i] = std::pow(theta, -double(i) / (kAttnD / 2));
    made_for = theta;
  }
  auto launch = [&](auto* type) {
    using T = std::remove_pointer_t<decltype(type)>;
    const T* x = static_cast<const T*>(qkv);
    T *q = static_cast<T*>(q_out), *k = static_cast<T*>(kcache), *v = static_cast<T*>(vcache);
    void* params[] = {&x, &row_stride, &q, &k, &v, &slots, &positions, &hq, &hkv, &page, &pages, &f};
    B200_CUDA_CHECK(launch_maybe_pdl(reinterpret_cast<const void*>(&rope_paged_append_kernel<T>), dim3(unsigned(rows)), dim3(kAppThreads), params, 0, stream, true));
  };
  if (t == DType::F16) launch(static_cast<__half*>(nullptr));
  else launch(static_cast<__nv_bfloat16*>(nullptr));
}

}  // namespace b200ipc
