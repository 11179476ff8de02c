// The parts of a split source, put together.
//
// Each part holds a row's normalised O_s and lse_s. With M the largest lse_s,
//   O = sum_s exp(lse_s - M) O_s / sum_s exp(lse_s - M),
//   lse = M + log sum_s exp(lse_s - M).
// A part without keys has lse -inf and adds nothing. A part with a NaN score has lse
// NaN, which the maximum passes over and its exponential brings into the sums: the
// parts are left out only where the lse of every one of them is -inf. W warps a row
// (four for many parts, whose reads would follow one another otherwise), four columns
// a lane.
#include <cmath>

#include "cross_attention.cuh"

namespace magma {
namespace {

constexpr int kThreads = 256;
// Parts beyond which four warps share a row: 8 x 32 heads over 8 of 128, 8192 keys, 32
// parts, 55 us (one warp a row 62); 8 heads, 100000 keys, 261 parts, 82 us (142); with few
// parts the warps have too little each: 64 x 32 heads over 8, 4096 keys, 5 parts, 166 us
// (four warps 169).
constexpr int kManyParts = 8;

template <typename T, int W>
__global__ void __launch_bounds__(kThreads)
cross_join(const float* __restrict__ part, const float* __restrict__ part_lse, T* __restrict__ o,
           float* __restrict__ lse, const CrossGeom g, int n_part) {
  constexpr int kRows = kThreads / 32 / W;
  __shared__ float4 sums[W > 1 ? kThreads : 1];
  __shared__ float totals[W > 1 ? kThreads / 32 : 1];
  wait_for_launch_before();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w = warp % W;
  const int64_t rows = g.batch * g.heads * g.q_len;
  const int64_t i = (int64_t)blockIdx.x * kRows + warp / W;
  const bool row_on = i < rows;
  float m = -INFINITY;
  bool some = false;  // a part that is not empty
  if (row_on)
    for (int s = lane; s < n_part; s += 32) {
      const float x = part_lse[s * rows + i];
      some = some || x != -INFINITY;
      m = fmaxf(m, x);
    }
  m = warp_max(m);
  some = __any_sync(0xffffffffu, some);
  float total = 0.f;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  const int c = lane * 4;
  if (some) {
    const int s0 = n_part * w / W, s1 = n_part * (w + 1) / W;
#pragma unroll 8
    for (int s = s0; s < s1; ++s) {
      const float f = expf(part_lse[s * rows + i] - m);
      total += f;
      if (c >= g.hd) continue;
      float v[4];
      load4(part + (s * rows + i) * g.hd + c, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(f, v[e], acc[e]);
    }
  }
  if constexpr (W > 1) {
    sums[threadIdx.x] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    if (lane == 0) totals[warp] = total;
    __syncthreads();
    if (w != 0) return;
#pragma unroll
    for (int x = 1; x < W; ++x) {
      const float4 v = sums[threadIdx.x + 32 * x];
      acc[0] += v.x, acc[1] += v.y, acc[2] += v.z, acc[3] += v.w;
      total += totals[warp + x];
    }
  }
  if (!row_on) return;
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const int64_t q = i % g.q_len, bh = i / g.q_len, h = bh % g.heads, b = bh / g.heads;
  if (c < g.hd) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= inv;
    store4(o + b * g.os[0] + h * g.os[1] + q * g.os[2] + c, acc);
  }
  if (lane == 0 && lse != nullptr) lse[i] = total == 0.f ? -INFINITY : m + logf(total);
}

template <typename T>
magma_status_t join(const float* part, const float* part_lse, void* o, float* lse,
                    const CrossGeom& g, int n_part, cudaStream_t s) {
  const int64_t rows = g.batch * g.heads * g.q_len;
  const bool many = n_part > kManyParts;
  const unsigned blocks = (unsigned)ceil_div(rows, many ? 2 : 8);
  return launch_after(many ? cross_join<T, 4> : cross_join<T, 1>, dim3(blocks), kThreads, 0, s,
                      "cross_join", part, part_lse, static_cast<T*>(o), lse, g, n_part);
}

}  // namespace

magma_status_t cross_join_parts(const float* part, const float* part_lse, void* o, float* lse,
                                const CrossGeom& g, int n_part, magma_dtype_t dtype,
                                cudaStream_t s) {
  return dtype == MAGMA_DTYPE_F32 ? join<float>(part, part_lse, o, lse, g, n_part, s)
                                  : join<__nv_bfloat16>(part, part_lse, o, lse, g, n_part, s);
}

}  // namespace magma
