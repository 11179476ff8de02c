// The parts of a split source, put together.
//
// Each part holds a row's normalised O_s and lse_s. With M the largest lse_s,
//   O = sum_s exp(lse_s - M) O_s / sum_s exp(lse_s - M),
//   lse = M + log sum_s exp(lse_s - M).
// A part without keys has lse -inf and is not read. One warp a row, four columns
// a lane; the parts of a few rows come out of L2.
#include <cmath>

#include "cross_attention.cuh"

namespace magma {
namespace {

template <typename T>
__global__ void __launch_bounds__(256)
cross_join(const float* __restrict__ part, const float* __restrict__ part_lse, T* __restrict__ o,
           float* __restrict__ lse, const CrossGeom g, int n_part) {
  wait_for_launch_before();
  const int lane = threadIdx.x & 31;
  const int64_t rows = g.batch * g.heads * g.q_len;
  const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= rows) return;
  float m = -INFINITY;
  for (int s = lane; s < n_part; s += 32) m = fmaxf(m, part_lse[s * rows + i]);
  m = warp_max(m);
  float total = 0.f;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  const int c = lane * 4;
  if (m != -INFINITY) {
#pragma unroll 4
    for (int s = 0; s < n_part; ++s) {
      const float w = expf(part_lse[s * rows + i] - m);
      total += w;
      if (c >= g.hd) continue;
      float v[4];
      load4(part + (s * rows + i) * g.hd + c, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(w, v[e], acc[e]);
    }
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const int64_t q = i % g.q_len, bh = i / g.q_len, h = bh % g.heads, b = bh / g.heads;
  if (c < g.hd) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= inv;
    store4(o + b * g.os[0] + h * g.os[1] + q * g.os[2] + c, acc);
  }
  if (lane == 0 && lse != nullptr) lse[i] = total == 0.f ? -INFINITY : m + logf(total);
}

}  // namespace

magma_status_t cross_join_parts(const float* part, const float* part_lse, void* o, float* lse,
                                const CrossGeom& g, int n_part, magma_dtype_t dtype,
                                cudaStream_t s) {
  const unsigned blocks = (unsigned)ceil_div(g.batch * g.heads * g.q_len, 8);
  if (dtype == MAGMA_DTYPE_F32)
    return launch_after(cross_join<float>, dim3(blocks), 256, 0, s, "cross_join", part, part_lse,
                        static_cast<float*>(o), lse, g, n_part);
  return launch_after(cross_join<__nv_bfloat16>, dim3(blocks), 256, 0, s, "cross_join", part, part_lse,
                      static_cast<__nv_bfloat16*>(o), lse, g, n_part);
}

}  // namespace magma
