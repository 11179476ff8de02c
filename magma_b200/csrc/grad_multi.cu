// Global gradient norm over many tensors, and clipping by it.
//
// optim.clipGradNorm (Sources/Core/Optimizer.swift:1229-1267) over the
// gradients of separately held parameters:
//   norm = sqrt(sum_i sum_e (g_i[e] * grad_scale)^2)
//   c    = max_norm / (norm + 1e-6) where that is below 1, else 1 (also for NaN)
//   out_i[e] = (g_i[e] * grad_scale) * c
// Two launches whatever the number of tensors (up to kBigList of them):
//   grad_multi_sumsq  every block adds the squares of its share of the list
//                     and writes one partial sum;
//   grad_multi_scale  every block adds all partial sums in the same order,
//                     forms c, and scales its share; block 0 writes the norm.
// The list travels in the kernel's parameters, so a captured graph holds its
// own copy and nothing is uploaded. The concatenated list is cut into
// kTile-element tiles (a tile never spans two tensors), which the blocks take
// in turn, so that the GPU reads one front through memory; one binary search
// finds a block's first tensor, and from there it walks along the list.
//
// The squares are added in 64 bits: a square of an F32 value neither overflows
// nor vanishes there, and the order of the additions does not show in the F32
// result. The products g * grad_scale and (..) * c are F32, as the reference's
// are; a BF16 output rounds once, from the F32 product.
//
// Bound by HBM: two reads and a write, since the factor needs all gradients first
// (225 tensors, 234 million F32 values: 135 + 306 us, 6.4 TB/s for the 2.8 GB), and by
// the two launches for a small model (407 KB in 4 tensors: 5 to 6 us).
#include <algorithm>
#include <new>
#include <vector>

#include "common.cuh"
#include "memory_views.cuh"

namespace magma {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 4096;       // elements of a tile
constexpr int kSmallList = 48;    // tensors per launch, parameters of about 1 KB,
constexpr int kMidList = 256;     // 7 KB
constexpr int kBigList = 1024;    // and 29 KB (the limit is 32764 bytes)
constexpr int kBlocksPerSm = 8;

template <int N>
struct GradList {
  const void* g[N];
  void* out[N];
  int64_t n[N];
  uint32_t first[N + 1];  // index of a tensor's first tile; first[count] = all tiles
  uint8_t kind[N];        // 1: g is BF16, 2: out is BF16, 4: vectors of four are aligned
  int count;
};

constexpr int kKindBf16In = 1, kKindBf16Out = 2, kKindVec = 4;

// The tensor that holds tile t.
template <int N>
__device__ __forceinline__ int tensor_of(const GradList<N>& l, uint32_t t) {
  int lo = 0, hi = l.count;  // first[lo] <= t < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (l.first[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Sum over the block's threads in a fixed order, valid in every thread.
__device__ __forceinline__ double block_sum(double x, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) t += red[i];
  return t;
}

template <typename T>
__device__ __forceinline__ double tile_sumsq(const T* g, int n, bool vec, float scale) {
  double acc = 0.0;
  constexpr int kPer = kTile / kThreads / 4;
  if (vec && n == kTile) {
    float v[kPer][4];
#pragma unroll
    for (int i = 0; i < kPer; ++i) load4(g + 4 * (threadIdx.x + i * kThreads), v[i]);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const double x = (double)__fmul_rn(v[i][e], scale);
        acc = fma(x, x, acc);
      }
  } else {
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const double x = (double)__fmul_rn(to_f32(g[i]), scale);
      acc = fma(x, x, acc);
    }
  }
  return acc;
}

template <int N>
__global__ void __launch_bounds__(kThreads)
grad_multi_sumsq(const __grid_constant__ GradList<N> l, float scale,
                 double* __restrict__ partial) {
  __shared__ double red[kThreads / 32];
  const uint32_t tiles = l.first[l.count];
  double acc = 0.0;
  if (blockIdx.x < tiles) {
    int k = tensor_of(l, blockIdx.x);
    for (uint32_t t = blockIdx.x; t < tiles; t += gridDim.x) {
      while (t >= l.first[k + 1]) ++k;
      const int64_t e0 = (int64_t)(t - l.first[k]) * kTile;
      const int64_t left = l.n[k] - e0;
      const int n = left < kTile ? (int)left : kTile;
      const bool vec = (l.kind[k] & kKindVec) != 0;
      acc += (l.kind[k] & kKindBf16In)
                 ? tile_sumsq(static_cast<const __nv_bfloat16*>(l.g[k]) + e0, n, vec, scale)
                 : tile_sumsq(static_cast<const float*>(l.g[k]) + e0, n, vec, scale);
    }
  }
  const double t = block_sum(acc, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = t;
}

// sqrt of all partial sums, the same double in every thread of every block.
__device__ __forceinline__ float norm_of(const double* partial, int nb, double* red) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < nb; i += kThreads) acc += partial[i];
  return (float)sqrt(block_sum(acc, red));
}

__global__ void __launch_bounds__(kThreads)
grad_multi_finish(const double* __restrict__ partial, int nb, float* __restrict__ norm) {
  __shared__ double red[kThreads / 32];
  wait_for_launch_before();
  const float v = norm_of(partial, nb, red);
  if (threadIdx.x == 0) norm[0] = v;
}

// Outputs are not read again here: they need not push gradients out of the L2.
__device__ __forceinline__ void stream4(float* p, const float (&v)[4]) {
  __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
}
__device__ __forceinline__ void stream4(__nv_bfloat16* p, const float (&v)[4]) {
  uint2 u;
  *reinterpret_cast<__nv_bfloat162*>(&u.x) = __floats2bfloat162_rn(v[0], v[1]);
  *reinterpret_cast<__nv_bfloat162*>(&u.y) = __floats2bfloat162_rn(v[2], v[3]);
  __stcs(reinterpret_cast<uint2*>(p), u);
}

template <typename TI, typename TO>
__device__ __forceinline__ void tile_scale(const TI* g, TO* out, int n, bool vec, float scale,
                                           float c) {
  constexpr int kPer = kTile / kThreads / 4;
  if (vec && n == kTile) {
    float v[kPer][4];
#pragma unroll
    for (int i = 0; i < kPer; ++i) load4(g + 4 * (threadIdx.x + i * kThreads), v[i]);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] = __fmul_rn(__fmul_rn(v[i][e], scale), c);
      stream4(out + 4 * (threadIdx.x + i * kThreads), v[i]);
    }
  } else {
    for (int i = threadIdx.x; i < n; i += kThreads)
      out[i] = from_f32<TO>(__fmul_rn(__fmul_rn(to_f32(g[i]), scale), c));
  }
}

// The list is walked backwards: what grad_multi_sumsq read last is what the L2
// still holds.
template <int N>
__global__ void __launch_bounds__(kThreads)
grad_multi_scale(const __grid_constant__ GradList<N> l, float scale, float max_norm,
                 const double* __restrict__ partial, int nb, float* __restrict__ norm) {
  __shared__ double red[kThreads / 32];
  wait_for_launch_before();
  const float v = norm_of(partial, nb, red);
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = v;
  const float raw = __fdiv_rn(max_norm, __fadd_rn(v, 1e-6f));
  const float c = raw < 1.f ? raw : 1.f;
  const uint32_t tiles = l.first[l.count];
  if (blockIdx.x >= tiles) return;
  int k = tensor_of(l, tiles - 1 - blockIdx.x);
  for (int64_t at = (int64_t)tiles - 1 - blockIdx.x; at >= 0; at -= gridDim.x) {
    const uint32_t t = (uint32_t)at;
    while (t < l.first[k]) --k;
    if (l.g[k] == l.out[k] && scale == 1.f && c == 1.f) continue;  // in place, unchanged
    const int64_t e0 = (int64_t)(t - l.first[k]) * kTile;
    const int64_t left = l.n[k] - e0;
    const int n = left < kTile ? (int)left : kTile;
    const bool vec = (l.kind[k] & kKindVec) != 0;
    const float* gf = static_cast<const float*>(l.g[k]) + e0;
    const __nv_bfloat16* gb = static_cast<const __nv_bfloat16*>(l.g[k]) + e0;
    float* of = static_cast<float*>(l.out[k]) + e0;
    __nv_bfloat16* ob = static_cast<__nv_bfloat16*>(l.out[k]) + e0;
    switch (l.kind[k] & (kKindBf16In | kKindBf16Out)) {
      case 0: tile_scale(gf, of, n, vec, scale, c); break;
      case kKindBf16In: tile_scale(gb, of, n, vec, scale, c); break;
      case kKindBf16Out: tile_scale(gf, ob, n, vec, scale, c); break;
      default: tile_scale(gb, ob, n, vec, scale, c); break;
    }
  }
}

struct Tensors {
  const void* const* g;
  void* const* out;  // NULL: norm only
  const int64_t* sizes;
  const magma_dtype_t* g_dtypes;
  const magma_dtype_t* out_dtypes;
  int32_t count;
};

bool vec_aligned(const void* p, magma_dtype_t t) {
  return (reinterpret_cast<uintptr_t>(p) & (4 * dtype_size(t) - 1)) == 0;
}

magma_status_t check(const char* fn, const Tensors& t) {
  MAGMA_REQUIRE(t.count >= 0, "%s: negative count", fn);
  if (t.count == 0) return MAGMA_OK;
  MAGMA_REQUIRE(t.g && t.sizes && t.g_dtypes, "%s: NULL array", fn);
  for (int32_t k = 0; k < t.count; ++k) {
    MAGMA_REQUIRE(t.sizes[k] >= 0 && t.sizes[k] < (1LL << 40), "%s: size %lld at %d", fn,
                  (long long)t.sizes[k], k);
    MAGMA_REQUIRE(is_float_dtype(t.g_dtypes[k]), "%s: gradient %d must be F32 or BF16", fn, k);
    MAGMA_REQUIRE(!t.out || is_float_dtype(t.out_dtypes[k]), "%s: output %d must be F32 or BF16",
                  fn, k);
    if (t.sizes[k] == 0) continue;
    MAGMA_REQUIRE(t.g[k] && (!t.out || t.out[k]), "%s: NULL tensor at %d", fn, k);
    MAGMA_REQUIRE(on_element(t.g[k], dtype_size(t.g_dtypes[k])) &&
                      (!t.out || on_element(t.out[k], dtype_size(t.out_dtypes[k]))),
                  "%s: tensor %d is not aligned to its element size", fn, k);
  }
  return MAGMA_OK;
}

// An output may be its own gradient (same address and dtype); otherwise it may
// share no memory with any other tensor of the call, the norm among them, which
// another block reads or writes at the same time.
magma_status_t check_overlap(const char* fn, const Tensors& t, const float* norm) {
  struct Range {
    uintptr_t begin, end;
    bool out;
  };
  std::vector<Range> r;
  r.reserve(2 * (size_t)t.count + 1);
  const uintptr_t n = reinterpret_cast<uintptr_t>(norm);
  r.push_back({n, n + sizeof(float), true});
  for (int32_t k = 0; k < t.count; ++k) {
    if (t.sizes[k] == 0) continue;
    const uintptr_t g = reinterpret_cast<uintptr_t>(t.g[k]);
    const uintptr_t o = reinterpret_cast<uintptr_t>(t.out[k]);
    r.push_back({o, o + t.sizes[k] * dtype_size(t.out_dtypes[k]), true});
    if (g != o || t.g_dtypes[k] != t.out_dtypes[k])
      r.push_back({g, g + t.sizes[k] * dtype_size(t.g_dtypes[k]), false});
  }
  std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
  uintptr_t end_any = 0, end_out = 0;
  for (const Range& x : r) {
    MAGMA_REQUIRE(x.begin >= (x.out ? end_any : end_out),
                  "%s: an output shares memory with another tensor of the list", fn);
    end_any = std::max(end_any, x.end);
    if (x.out) end_out = std::max(end_out, x.end);
  }
  return MAGMA_OK;
}

// Tensors k.. of the call into one list; returns the next tensor.
template <int N>
int32_t fill(const Tensors& t, int32_t k, GradList<N>* l) {
  l->count = 0;
  int64_t tiles = 0;
  for (; k < t.count && l->count < N; ++k) {
    if (t.sizes[k] == 0) continue;
    const int64_t more = ceil_div(t.sizes[k], kTile);
    if (tiles + more > 0x7FFFFFFFLL && l->count > 0) break;
    const int i = l->count++;
    l->g[i] = t.g[k];
    l->out[i] = t.out ? t.out[k] : nullptr;
    l->n[i] = t.sizes[k];
    l->first[i] = (uint32_t)tiles;
    tiles += more;
    bool vec = vec_aligned(t.g[k], t.g_dtypes[k]);
    int kind = t.g_dtypes[k] == MAGMA_DTYPE_BF16 ? kKindBf16In : 0;
    if (t.out) {
      vec = vec && vec_aligned(t.out[k], t.out_dtypes[k]);
      if (t.out_dtypes[k] == MAGMA_DTYPE_BF16) kind |= kKindBf16Out;
    }
    l->kind[i] = (uint8_t)(kind | (vec ? kKindVec : 0));
  }
  l->first[l->count] = (uint32_t)tiles;
  return k;
}

int blocks_for(uint32_t tiles) {
  const int64_t cap = (int64_t)kBlocksPerSm * num_sms();
  return (int)std::min<int64_t>(tiles, cap);
}

// Both passes over the call's lists, N tensors per launch.
template <int N>
magma_status_t run_lists(const char* fn, const Tensors& t, float grad_scale, float max_norm,
                         float* norm, double* partial, int64_t max_partial, cudaStream_t cs) {
  GradList<N> l;
  int nb = 0;
  for (int32_t k = 0; k < t.count;) {
    k = fill(t, k, &l);
    if (l.count == 0) continue;
    const int b = blocks_for(l.first[l.count]);
    MAGMA_REQUIRE(nb + b <= max_partial, "%s: workspace of magma_grad_norm_multi_workspace_size(%d) bytes needed",
                  fn, (int)t.count);
    grad_multi_sumsq<N><<<b, kThreads, 0, cs>>>(l, grad_scale, partial + nb);
    if (magma_status_t st = check_launch("grad_multi_sumsq")) return st;
    nb += b;
  }
  if (t.out == nullptr || nb == 0) {
    return launch_after(grad_multi_finish, dim3(1), kThreads, 0, cs, "grad_multi_finish", partial, nb,
                        norm);
  }
  bool first = true;
  for (int32_t k = 0; k < t.count;) {
    k = fill(t, k, &l);
    if (l.count == 0) continue;
    if (magma_status_t st = launch_after(grad_multi_scale<N>, dim3(blocks_for(l.first[l.count])),
                                         kThreads, 0, cs, "grad_multi_scale", l, grad_scale, max_norm,
                                         partial, nb, first ? norm : nullptr))
      return st;
    first = false;
  }
  return MAGMA_OK;
}

magma_status_t run(const char* fn, const Tensors& t, float grad_scale, float max_norm, float* norm,
                   void* workspace, int64_t workspace_bytes, void* stream) {
  if (magma_status_t st = check(fn, t)) return st;
  MAGMA_REQUIRE(norm != nullptr && on_element(norm, sizeof(float)),
                "%s: NULL norm, or one off its element", fn);
  MAGMA_REQUIRE(workspace != nullptr && workspace_bytes >= 0 &&
                    (reinterpret_cast<uintptr_t>(workspace) & 7u) == 0,
                "%s: an 8-byte aligned workspace is needed", fn);
  if (t.out) {
    try {
      if (magma_status_t st = check_overlap(fn, t, norm)) return st;
    } catch (const std::bad_alloc&) {
      return fail(MAGMA_RESOURCE_EXHAUSTED, "%s: out of host memory", fn);
    }
  }
  double* partial = static_cast<double*>(workspace);
  cudaStream_t cs = (cudaStream_t)stream;
  return t.count <= kSmallList
             ? run_lists<kSmallList>(fn, t, grad_scale, max_norm, norm, partial,
                                     workspace_bytes / 8, cs)
         : t.count <= kMidList
             ? run_lists<kMidList>(fn, t, grad_scale, max_norm, norm, partial, workspace_bytes / 8, cs)
             : run_lists<kBigList>(fn, t, grad_scale, max_norm, norm, partial,
                                   workspace_bytes / 8, cs);
}

}  // namespace
}  // namespace magma

using namespace magma;

extern "C" {

int64_t magma_grad_norm_multi_workspace_size(int32_t count) {
  const int64_t lists = count > 0 ? ceil_div(count, kBigList) : 1;
  return 8 * lists * kBlocksPerSm * num_sms();
}

magma_status_t magma_grad_norm_multi(const void* const* grads, const int64_t* sizes,
                                     const magma_dtype_t* dtypes, int32_t count, float grad_scale,
                                     float* norm, void* workspace, int64_t workspace_bytes,
                                     void* stream) {
  return run("magma_grad_norm_multi", Tensors{grads, nullptr, sizes, dtypes, nullptr, count},
             grad_scale, 0.f, norm, workspace, workspace_bytes, stream);
}

magma_status_t magma_clip_grad_norm_multi(const void* const* grads, void* const* out,
                                          const int64_t* sizes, const magma_dtype_t* grad_dtypes,
                                          const magma_dtype_t* out_dtypes, int32_t count,
                                          float grad_scale, float max_norm, float* norm,
                                          void* workspace, int64_t workspace_bytes, void* stream) {
  MAGMA_REQUIRE(max_norm > 0.f, "magma_clip_grad_norm_multi: max_norm must be positive");
  MAGMA_REQUIRE(count <= 0 || (out && out_dtypes), "magma_clip_grad_norm_multi: NULL array");
  return run("magma_clip_grad_norm_multi", Tensors{grads, out, sizes, grad_dtypes, out_dtypes, count},
             grad_scale, max_norm, norm, workspace, workspace_bytes, stream);
}

}  // extern "C"
