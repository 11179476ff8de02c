// Attention of queries over the keys and values of another sequence, F32 on
// the FMA pipe: F32 tensors, and BF16 tensors whose strides or head size the
// tensor-core kernels do not take.
//
//   S = scale Q K^T over the keys j < len_b;  P = softmax(S);  O = P V;
//   lse = log sum exp S.   A row without keys: O = 0, lse = -inf.
//   dV = P^T dO;  dS = P (dO V^T - delta), delta = rowsum(dO O);
//   dQ = scale dS K;  dK = scale dS^T Q;  dK and dV are summed over the query
//   heads that share a key head, by the CTA that owns the key tile.
//
// (nn.scaledDotProductAttention and MultiheadAttention, Sources/Core/
// Module.swift:2408-2441,2456-2660; VJP chain Sources/Core/Autodiff.swift:
// 309-317,379-386.) One pass over the keys with the running maximum and sum;
// every output element is added up by one thread in a fixed order. Keys from
// len_b on are never read: their tiles are filled with zeros.
//
// 64 x 64 tiles, 256 threads; thread (ty, tx) = (tid / 16, tid % 16) owns rows
// ty + 16i and columns tx + 16j.
#include <cmath>

#include "cross_attention.cuh"

namespace magma {
namespace {

constexpr int kT = 64;
constexpr int kThreads = 256;

// Rows [r0, r0 + 64) x [0, hd) of a head as F32 into dst[64][HD + 1], zeros
// from row `rows` and column hd on.
template <int HD, typename T>
__device__ __forceinline__ void load_tile(float* dst, const T* src, int64_t stride, int64_t r0,
                                          int64_t rows, int hd) {
  for (int i = threadIdx.x; i < kT * HD; i += kThreads) {
    const int r = i / HD, d = i % HD;
    dst[r * (HD + 1) + d] =
        r0 + r < rows && d < hd ? to_f32(src[(r0 + r) * stride + d]) : 0.f;
  }
}

// acc[i][j] += sum_d a[ty + 16i][d] * b[tx + 16j][d]
template <int HD>
__device__ __forceinline__ void dot_tile(float (&acc)[4][4], const float* a, const float* b,
                                         int ty, int tx) {
#pragma unroll 4
  for (int d = 0; d < HD; ++d) {
    float x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[(ty + 16 * i) * (HD + 1) + d];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = b[(tx + 16 * j) * (HD + 1) + d];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
  }
}

struct Block {
  int64_t tile, h, b;
};
__device__ __forceinline__ Block block_of(int64_t tiles, int64_t heads) {
  Block x;
  const int64_t i = blockIdx.x;
  x.tile = i % tiles;
  x.h = i / tiles % heads;
  x.b = i / tiles / heads;
  return x;
}

template <int HD, typename T>
__global__ void __launch_bounds__(kThreads)
cross_fwd(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
          T* __restrict__ o, float* __restrict__ lse, const CrossGeom g) {
  extern __shared__ float sm[];
  float* Qs = sm;
  float* Ks = Qs + kT * (HD + 1);
  float* Vs = Ks + kT * (HD + 1);
  float* Ps = Vs + kT * (HD + 1);  // [64][65]
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const Block x = block_of((g.q_len + kT - 1) / kT, g.heads);
  const int64_t q0 = x.tile * kT, kvh = x.h / g.group, len = cross_len(g, x.b);
  const T* kh = k + x.b * g.ks[0] + kvh * g.ks[1];
  const T* vh = v + x.b * g.vs[0] + kvh * g.vs[1];
  load_tile<HD>(Qs, q + x.b * g.qs[0] + x.h * g.qs[1], g.qs[2], q0, g.q_len, g.hd);
  constexpr int DJ = HD / 16;
  float acc[4][DJ] = {}, m[4], l[4] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = -INFINITY;
  for (int64_t k0 = 0; k0 < len; k0 += kT) {
    __syncthreads();
    load_tile<HD>(Ks, kh, g.ks[2], k0, len, g.hd);
    load_tile<HD>(Vs, vh, g.vs[2], k0, len, g.hd);
    __syncthreads();
    float s[4][4] = {};
    dot_tile<HD>(s, Qs, Ks, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = k0 + tx + 16 * j < len ? s[i][j] * g.scale : -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
      const float mn = fmaxf(m[i], mx);
      const float ref = mn == -INFINITY ? 0.f : mn;  // a row of -inf scores
      const float alpha = expf(m[i] - ref);
      float rs = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = expf(s[i][j] - ref);
        rs += s[i][j];
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) rs += __shfl_xor_sync(0xffffffffu, rs, w);
      l[i] = l[i] * alpha + rs;
      m[i] = mn;
#pragma unroll
      for (int j = 0; j < DJ; ++j) acc[i][j] *= alpha;
#pragma unroll
      for (int j = 0; j < 4; ++j) Ps[(ty + 16 * i) * (kT + 1) + tx + 16 * j] = s[i][j];
    }
    __syncthreads();
#pragma unroll 4
    for (int c = 0; c < kT; ++c) {
      float pv[4], vv[DJ];
#pragma unroll
      for (int i = 0; i < 4; ++i) pv[i] = Ps[(ty + 16 * i) * (kT + 1) + c];
#pragma unroll
      for (int j = 0; j < DJ; ++j) vv[j] = Vs[c * (HD + 1) + tx + 16 * j];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < DJ; ++j) acc[i][j] = fmaf(pv[i], vv[j], acc[i][j]);
    }
  }
  T* oh = o + x.b * g.os[0] + x.h * g.os[1];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t qi = q0 + ty + 16 * i;
    if (qi >= g.q_len) continue;
    const float inv = l[i] == 0.f ? 0.f : 1.0f / l[i];  // no keys: a zero row
#pragma unroll
    for (int j = 0; j < DJ; ++j) {
      const int d = tx + 16 * j;
      if (d < g.hd) oh[qi * g.os[2] + d] = from_f32<T>(acc[i][j] * inv);
    }
    if (tx == 0 && lse != nullptr)
      lse[(x.b * g.heads + x.h) * g.q_len + qi] = l[i] == 0.f ? -INFINITY : m[i] + logf(l[i]);
  }
}

// delta[b, h, i] = sum_d dO[i, d] * O[i, d]; one warp per row.
template <typename T>
__global__ void __launch_bounds__(kThreads)
cross_delta(const T* __restrict__ o, const T* __restrict__ d_o, float* __restrict__ delta,
            const CrossGeom g) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = g.batch * g.heads * g.q_len;
  for (int64_t r = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); r < rows;
       r += (int64_t)gridDim.x * (kThreads / 32)) {
    const int64_t s = r % g.q_len, bh = r / g.q_len, h = bh % g.heads, b = bh / g.heads;
    const T* po = o + b * g.os[0] + h * g.os[1] + s * g.os[2];
    const T* pd = d_o + b * g.dos[0] + h * g.dos[1] + s * g.dos[2];
    float acc = 0.f;
    for (int d = lane; d < g.hd; d += 32) acc = fmaf(to_f32(pd[d]), to_f32(po[d]), acc);
    acc = warp_sum(acc);
    if (lane == 0) delta[r] = acc;
  }
}

// A row without probabilities (lse = -inf) gets none in the gradient either.
__device__ __forceinline__ float row_lse(float lse) { return lse == -INFINITY ? INFINITY : lse; }

// P and dS of a 64 x 64 tile from its dot products; keys from len on and
// queries from q_len on take no part.
__device__ __forceinline__ void probs(float& s, float& dp, bool on, float scale, float lse,
                                      float delta) {
  const float p = on ? expf(s * scale - lse) : 0.f;
  s = p;
  dp = on ? p * (dp - delta) : 0.f;
}

// One CTA per (key tile, key head, sequence): dK and dV of 64 keys.
template <int HD, typename T>
__global__ void __launch_bounds__(kThreads)
cross_dkdv(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
           const T* __restrict__ d_o, const float* __restrict__ lse,
           const float* __restrict__ delta, T* __restrict__ dk, T* __restrict__ dv,
           const CrossGeom g) {
  extern __shared__ float sm[];
  float* Ks = sm;
  float* Vs = Ks + kT * (HD + 1);
  float* Qs = Vs + kT * (HD + 1);
  float* Gs = Qs + kT * (HD + 1);   // dO
  float* Ps = Gs + kT * (HD + 1);   // [q][k], 64 x 65
  float* Ds = Ps + kT * (kT + 1);   // dS
  float* Ls = Ds + kT * (kT + 1);   // lse of the query tile
  float* Es = Ls + kT;              // delta of the query tile
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const Block x = block_of((g.kv_len + kT - 1) / kT, g.kv_heads);
  const int64_t k0 = x.tile * kT, len = cross_len(g, x.b);
  constexpr int DJ = HD / 16;
  float adk[4][DJ] = {}, adv[4][DJ] = {};
  if (k0 < len) {
    load_tile<HD>(Ks, k + x.b * g.ks[0] + x.h * g.ks[1], g.ks[2], k0, len, g.hd);
    load_tile<HD>(Vs, v + x.b * g.vs[0] + x.h * g.vs[1], g.vs[2], k0, len, g.hd);
    for (int gi = 0; gi < g.group; ++gi) {
      const int64_t h = x.h * g.group + gi, bh = x.b * g.heads + h;
      const T* qh = q + x.b * g.qs[0] + h * g.qs[1];
      const T* doh = d_o + x.b * g.dos[0] + h * g.dos[1];
      for (int64_t q0 = 0; q0 < g.q_len; q0 += kT) {
        __syncthreads();
        load_tile<HD>(Qs, qh, g.qs[2], q0, g.q_len, g.hd);
        load_tile<HD>(Gs, doh, g.dos[2], q0, g.q_len, g.hd);
        if (tid < kT) {
          const bool on = q0 + tid < g.q_len;
          Ls[tid] = on ? row_lse(lse[bh * g.q_len + q0 + tid]) : 0.f;
          Es[tid] = on ? delta[bh * g.q_len + q0 + tid] : 0.f;
        }
        __syncthreads();
        float s[4][4] = {}, dp[4][4] = {};
        dot_tile<HD>(s, Qs, Ks, ty, tx);
        dot_tile<HD>(dp, Gs, Vs, ty, tx);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = ty + 16 * i, c = tx + 16 * j;
            probs(s[i][j], dp[i][j], k0 + c < len && q0 + r < g.q_len, g.scale, Ls[r], Es[r]);
            Ps[r * (kT + 1) + c] = s[i][j];
            Ds[r * (kT + 1) + c] = dp[i][j];
          }
        __syncthreads();
        // dV[key][d] += sum_q P[q][key] dO[q][d]: keys ty + 16i, columns tx + 16j
#pragma unroll 2
        for (int r = 0; r < kT; ++r) {
          float p[4], ds[4], qv[DJ], gv[DJ];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[i] = Ps[r * (kT + 1) + ty + 16 * i];
            ds[i] = Ds[r * (kT + 1) + ty + 16 * i];
          }
#pragma unroll
          for (int j = 0; j < DJ; ++j) {
            qv[j] = Qs[r * (HD + 1) + tx + 16 * j];
            gv[j] = Gs[r * (HD + 1) + tx + 16 * j];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < DJ; ++j) {
              adv[i][j] = fmaf(p[i], gv[j], adv[i][j]);
              adk[i][j] = fmaf(ds[i], qv[j], adk[i][j]);
            }
        }
      }
    }
  }
  T* dkh = dk + x.b * g.dks[0] + x.h * g.dks[1];
  T* dvh = dv + x.b * g.dvs[0] + x.h * g.dvs[1];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t kj = k0 + ty + 16 * i;
    if (kj >= g.kv_len) continue;
#pragma unroll
    for (int j = 0; j < DJ; ++j) {
      const int d = tx + 16 * j;
      if (d >= g.hd) continue;
      dkh[kj * g.dks[2] + d] = from_f32<T>(adk[i][j] * g.scale);
      dvh[kj * g.dvs[2] + d] = from_f32<T>(adv[i][j]);
    }
  }
}

// One CTA per (query tile, head, sequence): dQ of 64 queries.
template <int HD, typename T>
__global__ void __launch_bounds__(kThreads)
cross_dq(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
         const T* __restrict__ d_o, const float* __restrict__ lse,
         const float* __restrict__ delta, T* __restrict__ dq, const CrossGeom g) {
  extern __shared__ float sm[];
  float* Qs = sm;
  float* Gs = Qs + kT * (HD + 1);
  float* Ks = Gs + kT * (HD + 1);
  float* Vs = Ks + kT * (HD + 1);
  float* Ds = Vs + kT * (HD + 1);  // [q][k], 64 x 65
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const Block x = block_of((g.q_len + kT - 1) / kT, g.heads);
  const int64_t q0 = x.tile * kT, kvh = x.h / g.group, len = cross_len(g, x.b);
  const int64_t bh = x.b * g.heads + x.h;
  load_tile<HD>(Qs, q + x.b * g.qs[0] + x.h * g.qs[1], g.qs[2], q0, g.q_len, g.hd);
  load_tile<HD>(Gs, d_o + x.b * g.dos[0] + x.h * g.dos[1], g.dos[2], q0, g.q_len, g.hd);
  float ls[4], es[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t qi = q0 + ty + 16 * i;
    ls[i] = qi < g.q_len ? row_lse(lse[bh * g.q_len + qi]) : 0.f;
    es[i] = qi < g.q_len ? delta[bh * g.q_len + qi] : 0.f;
  }
  constexpr int DJ = HD / 16;
  float acc[4][DJ] = {};
  for (int64_t k0 = 0; k0 < len; k0 += kT) {
    __syncthreads();
    load_tile<HD>(Ks, k + x.b * g.ks[0] + kvh * g.ks[1], g.ks[2], k0, len, g.hd);
    load_tile<HD>(Vs, v + x.b * g.vs[0] + kvh * g.vs[1], g.vs[2], k0, len, g.hd);
    __syncthreads();
    float s[4][4] = {}, dp[4][4] = {};
    dot_tile<HD>(s, Qs, Ks, ty, tx);
    dot_tile<HD>(dp, Gs, Vs, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = ty + 16 * i, c = tx + 16 * j;
        probs(s[i][j], dp[i][j], k0 + c < len && q0 + r < g.q_len, g.scale, ls[i], es[i]);
        Ds[r * (kT + 1) + c] = dp[i][j];
      }
    __syncthreads();
#pragma unroll 4
    for (int c = 0; c < kT; ++c) {
      float ds[4], kv[DJ];
#pragma unroll
      for (int i = 0; i < 4; ++i) ds[i] = Ds[(ty + 16 * i) * (kT + 1) + c];
#pragma unroll
      for (int j = 0; j < DJ; ++j) kv[j] = Ks[c * (HD + 1) + tx + 16 * j];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < DJ; ++j) acc[i][j] = fmaf(ds[i], kv[j], acc[i][j]);
    }
  }
  T* dqh = dq + x.b * g.dqs[0] + x.h * g.dqs[1];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t qi = q0 + ty + 16 * i;
    if (qi >= g.q_len) continue;
#pragma unroll
    for (int j = 0; j < DJ; ++j) {
      const int d = tx + 16 * j;
      if (d < g.hd) dqh[qi * g.dqs[2] + d] = from_f32<T>(acc[i][j] * g.scale);
    }
  }
}

magma_status_t blocks_of(int64_t tiles, int64_t heads, int64_t batch, unsigned* n) {
  const double all = (double)tiles * (double)heads * (double)batch;
  if (all > 2147483647.0)
    return fail(MAGMA_INVALID_ARGUMENT, "cross attention: more than 2^31 - 1 tiles");
  *n = (unsigned)(tiles * heads * batch);
  return MAGMA_OK;
}

template <int HD, typename T>
magma_status_t fwd(const void* q, const void* k, const void* v, void* o, float* lse,
                   const CrossGeom& g, cudaStream_t s) {
  const size_t smem = (3 * kT * (HD + 1) + kT * (kT + 1)) * sizeof(float);
  unsigned n;
  if (magma_status_t st = cross_smem<cross_fwd<HD, T>>((int)smem)) return st;
  if (magma_status_t st = blocks_of(ceil_div(g.q_len, kT), g.heads, g.batch, &n)) return st;
  cross_fwd<HD, T><<<n, kThreads, smem, s>>>((const T*)q, (const T*)k, (const T*)v, (T*)o, lse, g);
  return check_launch("cross_fwd");
}

template <int HD, typename T>
magma_status_t bwd(const void* q, const void* k, const void* v, const void* o, const void* d_o,
                   const float* lse, void* dq, void* dk, void* dv, float* delta,
                   const CrossGeom& g, cudaStream_t s) {
  const size_t kv_smem =
      (4 * kT * (HD + 1) + 2 * kT * (kT + 1) + 2 * kT) * sizeof(float);
  const size_t q_smem = (4 * kT * (HD + 1) + kT * (kT + 1)) * sizeof(float);
  if (magma_status_t st = cross_smem<cross_dkdv<HD, T>>((int)kv_smem)) return st;
  if (magma_status_t st = cross_smem<cross_dq<HD, T>>((int)q_smem)) return st;
  unsigned nq = 0, nk = 0;
  if (magma_status_t st = blocks_of(ceil_div(g.q_len, kT), g.heads, g.batch, &nq)) return st;
  if (magma_status_t st = blocks_of(ceil_div(g.kv_len, kT), g.kv_heads, g.batch, &nk)) return st;
  if (nq > 0) {
    const int64_t rows = g.batch * g.heads * g.q_len;
    const int64_t cap = 16LL * num_sms();
    const int64_t nd = ceil_div(rows, kThreads / 32);
    cross_delta<T><<<(unsigned)(nd > cap ? cap : nd), kThreads, 0, s>>>((const T*)o, (const T*)d_o,
                                                                     delta, g);
    if (magma_status_t st = check_launch("cross_delta")) return st;
  }
  if (nk > 0) {
    cross_dkdv<HD, T><<<nk, kThreads, kv_smem, s>>>((const T*)q, (const T*)k, (const T*)v,
                                                    (const T*)d_o, lse, delta, (T*)dk, (T*)dv, g);
    if (magma_status_t st = check_launch("cross_dkdv")) return st;
  }
  if (nq > 0) {
    cross_dq<HD, T><<<nq, kThreads, q_smem, s>>>((const T*)q, (const T*)k, (const T*)v,
                                                 (const T*)d_o, lse, delta, (T*)dq, g);
    return check_launch("cross_dq");
  }
  return MAGMA_OK;
}

}  // namespace

magma_status_t cross_fwd_simt(const void* q, const void* k, const void* v, void* o, float* lse,
                              const CrossGeom& g, magma_dtype_t dtype, cudaStream_t s) {
  if (dtype == MAGMA_DTYPE_F32)
    return g.hd <= 64 ? fwd<64, float>(q, k, v, o, lse, g, s) : fwd<128, float>(q, k, v, o, lse, g, s);
  return g.hd <= 64 ? fwd<64, __nv_bfloat16>(q, k, v, o, lse, g, s)
                    : fwd<128, __nv_bfloat16>(q, k, v, o, lse, g, s);
}

magma_status_t cross_bwd_simt(const void* q, const void* k, const void* v, const void* o,
                              const void* d_o, const float* lse, void* dq, void* dk, void* dv,
                              float* delta, const CrossGeom& g, magma_dtype_t dtype,
                              cudaStream_t s) {
  if (dtype == MAGMA_DTYPE_F32)
    return g.hd <= 64 ? bwd<64, float>(q, k, v, o, d_o, lse, dq, dk, dv, delta, g, s)
                      : bwd<128, float>(q, k, v, o, d_o, lse, dq, dk, dv, delta, g, s);
  return g.hd <= 64 ? bwd<64, __nv_bfloat16>(q, k, v, o, d_o, lse, dq, dk, dv, delta, g, s)
                    : bwd<128, __nv_bfloat16>(q, k, v, o, d_o, lse, dq, dk, dv, delta, g, s);
}

}  // namespace magma
