// Embedding lookup with a scale and an optional position row, and its gradient
// by sorted tokens.
//
//   out[b*S + s, :]  = scale * table[tokens[b, s], :] + pos[s, :]
//   dtable[v, :] (+)= scale * sum_{r : tokens[r] = v, v != padding} dout[r, :]
//   dpos[s, :]   (+)= sum_b dout[b*S + s, :]
//
// (nn.Embedding, Sources/Core/Module.swift:339-410, with the sqrt(d) scale of
// encoder-decoder models; Data.swift:856-907.) F32 arithmetic, one rounding
// when a result is stored as BF16.
//
// Gradient, three launches:
//  1. emb_sort     one cluster of up to 8 CTAs sorts the rows by (token, row)
//                  with a stable radix sort, 8 bits a pass; rows whose token
//                  is padding or outside the table get the key `vocab` and
//                  end up last. The other clusters meanwhile set the table's
//                  gradient to zero and write dpos: neither needs the order,
//                  and the sort alone would leave 140 SMs idle. (The rows of
//                  tokens that occur are written twice.)
//  2. emb_sum      a CTA adds the dout rows of P consecutive places of the
//                  sorted order, so that every CTA has the same work however
//                  often a token repeats. A run of equal tokens inside the P
//                  places is stored at once; the part of a run that crosses a
//                  border goes to the workspace.
//  3. emb_join     adds the parts of each crossing run in order.
// The order of the additions depends on the tokens alone (no atomics on
// floating values), so the result is the same on every run.
//
// What bounds it (GPU time of the three launches): 32768 rows of 1024 BF16, 50257
// tokens: 35 + 16 + 9 us, the 206 MB of the table's F32 gradient and the 67 MB of
// dout at 4.6 TB/s; writing the zeros takes longer than the sort beside it. 16384
// rows of 384, 65 tokens: 10 + 9 + 8 us alone, 18 to 20 behind one another (a launch
// may begin before the one before it ends). That is not the 26 MB, which take 4 us, but a
// chain of trips to memory: the sort's one pass (counts, exchange in the cluster,
// places), then 32 places of a tile in four rounds of eight rows, then the parts of
// the runs; emb_sum has 12% of the warps that fit, emb_join issues in 13% of its cycles.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "memory_views.cuh"
#include "sm100.cuh"

namespace magma {
namespace {

namespace cg = cooperative_groups;

// ---- lookup --------------------------------------------------------------------
// A warp per row and pass of U vectors a lane, all loads of a pass first. 32 x 1024
// rows of 1024 F32 with the word frequencies of a text: 40 to 42 us. 9.9 thousand rows
// of the table occur, so HBM has to carry 179 MB (27 us); with the repeated table and
// position rows, which the L2 serves (46% of its reads hit), 405 MB pass through the
// SMs. DRAM is at 37% of its peak; the warps wait for their loads (26% of them fit, at
// 96 registers). 16 rows of 512 BF16: 2.1 us, a launch.
template <typename TI, typename TO, int V>
__global__ void __launch_bounds__(128)
emb_lookup(const int32_t* __restrict__ tokens, const TI* __restrict__ table, int64_t table_ld,
           const TI* __restrict__ pos, TO* __restrict__ out, int64_t rows, int64_t seq, int dim,
           int64_t vocab, float scale, int* err) {
  constexpr int U = V == 1 ? 8 : 4;
  const int lane = threadIdx.x & 31;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5); r < rows;
       r += (int64_t)gridDim.x * 4) {
    const int32_t t = tokens[r];
    const bool bad = t < 0 || t >= vocab;
    if (bad && lane == 0) set_device_error(err, kDevErrBadIndex);
    const TI* src = table + (bad ? 0 : (int64_t)t * table_ld);
    const TI* ps = pos ? pos + (r % seq) * dim : nullptr;
    TO* dst = out + r * dim;
    for (int c0 = 0; c0 < dim; c0 += 32 * V * U) {
      float a[U][V], p[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + (u * 32 + lane) * V;
        if (c >= dim) continue;
        if constexpr (V == 8) load8(src + c, a[u]);
        else a[u][0] = to_f32(src[c]);
        if (ps != nullptr) {
          if constexpr (V == 8) load8(ps + c, p[u]);
          else p[u][0] = to_f32(ps[c]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + (u * 32 + lane) * V;
        if (c >= dim) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float x = bad ? 0.f : __fmul_rn(a[u][e], scale);
          if (ps != nullptr) x = __fadd_rn(x, p[u][e]);
          a[u][e] = x;
        }
        if constexpr (V == 8) store8(dst + c, a[u]);
        else dst[c] = from_f32<TO>(a[u][0]);
      }
    }
  }
}

// ---- 16-byte accesses -----------------------------------------------------------
// V elements of T as they lie in memory, kept packed until they are added.
template <typename T, int V>
struct Raw {
  static constexpr int kWords = (V * (int)sizeof(T) + 3) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kWords == 4) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    } else if constexpr (sizeof(T) == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ void add_to(float (&acc)[V]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += __uint_as_float(w[e]);
    } else if constexpr (V == 1) {
      acc[0] += __uint_as_float(w[0] << 16);
    } else {
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        acc[e] += __uint_as_float(w[e / 2] << 16);
        acc[e + 1] += __uint_as_float(w[e / 2] & 0xFFFF0000u);
      }
    }
  }
};
template <typename T, int V>
__device__ __forceinline__ void load_v(const T* p, float (&v)[V]) {
  if constexpr (V == 8) load8(p, v);
  else if constexpr (V == 4) load4(p, v);
  else v[0] = to_f32(p[0]);
}
template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const float (&v)[V]) {
  if constexpr (V == 8) store8(p, v);
  else if constexpr (V == 4) store4(p, v);
  else p[0] = from_f32<T>(v[0]);
}

struct GradArgs {
  const int32_t* tokens;
  uint32_t* key[2];  // ping-pong buffers of the sort
  uint32_t* row[2];
  const void* dout;
  int64_t dout_ld;
  void* dtable;
  int64_t dtable_ld;
  float* head;  // [tile][dim]: the tile's part of a run that began before it
  float* tail;  // [tile][dim]: the tile's part of a run that began in it and goes on
  float* dpos;
  int64_t rows, vocab, batch, seq, padding, tiles;
  int dim, places, passes, accumulate, accumulate_dpos;
  float scale;
  int* err;
};

// ---- sort, zero rows, dpos ---------------------------------------------------------
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kDigits = 256;
constexpr int kCountBytes = kSortWarps * kDigits * 4;
// Rows up to which the cluster has one CTA; twice as many have two, and so on to eight.
// (64 columns, 65 tokens: 4096 rows 12.8 us, with 1024 here 11.6, with 4096 15.6; 16384
// rows of 384: 20.4, 20.3 and 24.0.)
constexpr int kSortRows = 2048;

__device__ __forceinline__ uint32_t sort_key(const GradArgs& a, int64_t i, bool report) {
  const int32_t t = a.tokens[i];
  if (t < 0 || t >= a.vocab) {
    if (report) set_device_error(a.err, kDevErrBadIndex);
    return (uint32_t)a.vocab;
  }
  return t == a.padding ? (uint32_t)a.vocab : (uint32_t)t;
}

// Every warp owns a contiguous piece of the rows. A pass counts the digits of
// each piece, turns the counts into the first place of (digit, CTA, warp) in
// that order, and moves the rows; within 32 rows the place follows the lane,
// so equal digits keep their order. All CTAs of the first cluster are here.
__device__ void sort_rows(const GradArgs& a, cg::cluster_group cluster, uint32_t* counts,
                          uint32_t* cta_count, uint32_t* scan) {
  const int nc = (int)cluster.num_blocks(), c = (int)cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t pieces = (int64_t)nc * kSortWarps;
  const int64_t piece = ((a.rows + pieces - 1) / pieces + 31) / 32 * 32;
  int64_t i0 = ((int64_t)c * kSortWarps + warp) * piece;
  int64_t i1 = i0 + piece;
  if (i0 > a.rows) i0 = a.rows;
  if (i1 > a.rows) i1 = a.rows;
  uint32_t* mine = counts + warp * kDigits;
  for (int p = 0; p < a.passes; ++p) {
    const int shift = 8 * p;
    const uint32_t* kin = p & 1 ? a.key[0] : a.key[1];
    const uint32_t* rin = p & 1 ? a.row[0] : a.row[1];
    uint32_t* kout = p & 1 ? a.key[1] : a.key[0];
    uint32_t* rout = p & 1 ? a.row[1] : a.row[0];
    for (int d = lane; d < kDigits; d += 32) mine[d] = 0;
    __syncwarp();
#pragma unroll 4
    for (int64_t i = i0 + lane; i < i1; i += 32) {
      const uint32_t k = p == 0 ? sort_key(a, i, true) : kin[i];
      atomicAdd(&mine[(k >> shift) & (kDigits - 1)], 1u);
    }
    __syncthreads();
    // counts[w][d] -> rows of digit d in earlier warps of this CTA
    if (threadIdx.x < kDigits) {
      uint32_t run = 0;
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t n = counts[w * kDigits + threadIdx.x];
        counts[w * kDigits + threadIdx.x] = run;
        run += n;
      }
      cta_count[threadIdx.x] = run;
    }
    cluster.sync();
    uint32_t before = 0, all = 0;  // rows of this digit in earlier CTAs, in all
    if (threadIdx.x < kDigits) {
#pragma unroll
      for (int o = 0; o < kMaxCluster; ++o) {
        const uint32_t n = o < nc ? cluster.map_shared_rank(cta_count, o)[threadIdx.x] : 0u;
        if (o < c) before += n;
        all += n;
      }
      scan[threadIdx.x] = all;
    }
    __syncthreads();
    if (warp == 0) {  // exclusive scan of the 256 totals
      uint32_t v[8], sum = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = scan[lane * 8 + e];
        sum += v[e];
      }
      uint32_t inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t n = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += n;
      }
      uint32_t run = inc - sum;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        scan[lane * 8 + e] = run;
        run += v[e];
      }
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
      const uint32_t base = scan[threadIdx.x] + before;
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) counts[w * kDigits + threadIdx.x] += base;
    }
    __syncthreads();
    for (int64_t j = i0; j < i1; j += 32) {
      const int64_t i = j + lane;
      const bool on = i < i1;
      const uint32_t active = __ballot_sync(0xffffffffu, on);
      if (on) {
        const uint32_t k = p == 0 ? sort_key(a, i, false) : kin[i];
        const uint32_t r = p == 0 ? (uint32_t)i : rin[i];
        const uint32_t d = (k >> shift) & (kDigits - 1);
        const uint32_t same = __match_any_sync(active, d);
        const uint32_t at = mine[d] + __popc(same & ((1u << lane) - 1));
        __syncwarp(active);
        if ((same >> lane) == 1u) mine[d] = at + 1;  // the last lane of this digit
        kout[at] = k;
        rout[at] = r;
      }
      __syncwarp();
    }
    // The next pass reads what the other CTAs wrote, and this CTA's counts are
    // read by them until here.
    if (p + 1 < a.passes) __threadfence();
    cluster.sync();
  }
}

// dpos: a thread has V columns of one position and every G-th stretch of the
// batch; the G sums of a column meet in shared memory and are added in order.
template <typename TD, int V>
__device__ void sum_positions(const GradArgs& a, int64_t cta, int64_t ctas, float* sums) {
  const int64_t nv = a.dim / V, items = a.seq * nv;
  // as many stretches as fill the CTAs, of at least eight rows
  int G = 1;
  while (G < 8 && items * G * 2 <= ctas * kSortThreads && a.batch >= G * 16) G *= 2;
  const int per = kSortThreads / G, g = threadIdx.x / per, x = threadIdx.x % per;
  const int64_t b0 = a.batch * g / G, b1 = a.batch * (g + 1) / G;
  const int64_t step = a.seq * a.dout_ld;
  for (int64_t i0 = cta * per; i0 < items; i0 += ctas * per) {
    const int64_t i = i0 + x, s = i / nv;
    const int col = (int)(i % nv) * V;
    float acc[V] = {};
    if (i < items) {
      const TD* src = static_cast<const TD*>(a.dout) + s * a.dout_ld + col;
      for (int64_t b = b0; b < b1; b += 8) {
        Raw<TD, V> v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (b + u < b1) v[u].load(src + (b + u) * step);
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (b + u < b1) v[u].add_to(acc);
      }
    }
    if (G > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < V; ++e) sums[e * kSortThreads + threadIdx.x] = acc[e];
      __syncthreads();
      if (g != 0) continue;
      for (int o = 1; o < G; ++o)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += sums[e * kSortThreads + o * per + x];
    }
    if (i >= items) continue;
    float* dst = a.dpos + s * a.dim + col;
    if (a.accumulate_dpos) {
      float old[V];
      load_v<float, V>(dst, old);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += old[e];
    }
    store_v<float, V>(dst, acc);
  }
}

template <typename TD, typename TT, int V>
__global__ void __launch_bounds__(kSortThreads, 1) emb_sort(const __grid_constant__ GradArgs a) {
  extern __shared__ __align__(128) uint32_t counts[];  // [warp][digit]
  __shared__ uint32_t cta_count[kDigits], scan[kDigits];
  cg::cluster_group cluster = cg::this_cluster();
  const int nc = (int)cluster.num_blocks();
  if ((int)blockIdx.x < nc) {
    if (a.rows > 0) sort_rows(a, cluster, counts, cta_count, scan);
    if ((int)gridDim.x > nc) return;  // the other clusters do the rest
  }
  const int64_t first = (int)gridDim.x > nc ? nc : 0;
  const int64_t cta = (int64_t)blockIdx.x - first, ctas = (int64_t)gridDim.x - first;
  __syncthreads();
  if (a.dpos != nullptr) sum_positions<TD, V>(a, cta, ctas, reinterpret_cast<float*>(counts));
  if (a.accumulate) return;
  TT* table = static_cast<TT*>(a.dtable);
  if constexpr (V > 1) {
    // Rows of whole 16-byte pieces: bulk copies of a zeroed stretch of shared
    // memory, 32 lanes issuing a row each.
    __syncthreads();
    uint4* z = reinterpret_cast<uint4*>(counts);
    for (int i = threadIdx.x; i < kCountBytes / 16; i += kSortThreads) z[i] = make_uint4(0, 0, 0, 0);
    sm100::fence_proxy_async_smem();
    __syncthreads();
    if (threadIdx.x >= 32) return;
    const uint32_t src = sm100::smem_u32(counts);
    const int64_t bytes = (int64_t)a.dim * sizeof(TT);
    for (int64_t v = cta * 32 + threadIdx.x; v < a.vocab; v += ctas * 32) {
      uint8_t* dst = reinterpret_cast<uint8_t*>(table + v * a.dtable_ld);
      for (int64_t at = 0; at < bytes; at += kCountBytes)
        sm100::bulk_store(dst + at, src,
                          (uint32_t)(bytes - at < kCountBytes ? bytes - at : kCountBytes));
    }
    sm100::bulk_commit_group();
    sm100::bulk_wait_group_all();
  } else {
    const int lane = threadIdx.x & 31;
    const int64_t w0 = (cta * kSortThreads + threadIdx.x) >> 5, warps = ctas * kSortWarps;
    for (int64_t v = w0; v < a.vocab; v += warps)
      for (int c = lane; c < a.dim; c += 32) table[v * a.dtable_ld + c] = from_f32<TT>(0.f);
  }
}

// ---- sum -----------------------------------------------------------------------
constexpr int kSumThreads = 128;
constexpr int kMaxPlaces = 128;

template <typename T, int V>
__device__ __forceinline__ void store_grad(const GradArgs& a, uint32_t token, int col,
                                           const float (&acc)[V]) {
  T* dst = static_cast<T*>(a.dtable) + (int64_t)token * a.dtable_ld + col;
  float v[V];
  if (a.accumulate) load_v<T, V>(dst, v);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float s = __fmul_rn(acc[e], a.scale);
    v[e] = a.accumulate ? __fadd_rn(v[e], s) : s;
  }
  store_v<T, V>(dst, v);
}

__device__ __forceinline__ const uint32_t* sorted_key(const GradArgs& a) {
  return a.passes & 1 ? a.key[0] : a.key[1];
}
__device__ __forceinline__ const uint32_t* sorted_row(const GradArgs& a) {
  return a.passes & 1 ? a.row[0] : a.row[1];
}

// TD: dout, TT: dtable. The dout rows of eight places are in flight at a time.
template <typename TD, typename TT, int V>
__global__ void __launch_bounds__(kSumThreads) emb_sum(const __grid_constant__ GradArgs a) {
  __shared__ uint32_t key[kMaxPlaces + 2], row[kMaxPlaces];
  wait_for_launch_before();
  const int64_t tile = blockIdx.x, p0 = tile * a.places;
  const int n = (int)(a.rows - p0 < a.places ? a.rows - p0 : a.places);
  const uint32_t* skey = sorted_key(a);
  const uint32_t* srow = sorted_row(a);
  // key[0]: the place before the tile, key[n + 1]: the place behind it
  for (int i = threadIdx.x; i < n + 2; i += kSumThreads) {
    const int64_t p = p0 + i - 1;
    key[i] = p >= 0 && p < a.rows ? skey[p] : 0xFFFFFFFFu;
    if (i >= 1 && i <= n) row[i - 1] = srow[p];
  }
  __syncthreads();
  const int col = (blockIdx.y * kSumThreads + threadIdx.x) * V;
  if (col >= a.dim) return;
  const TD* src = static_cast<const TD*>(a.dout) + col;
  float acc[V] = {};
  bool began = key[0] != key[1];  // the current run begins in this tile
  constexpr int kAhead = 8;
  for (int i0 = 0; i0 < n; i0 += kAhead) {
    Raw<TD, V> v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (i0 + u < n && key[i0 + u + 1] < (uint32_t)a.vocab)
        v[u].load(src + (int64_t)row[i0 + u] * a.dout_ld);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u;
      if (i >= n) break;
      const uint32_t t = key[i + 1];
      if (t >= (uint32_t)a.vocab) return;  // padding and bad tokens are last
      v[u].add_to(acc);
      const bool ends = key[i + 2] != t;
      if (!ends && i + 1 < n) continue;
      if (began && ends) {
        store_grad<TT, V>(a, t, col, acc);
      } else {
        float* part = (began ? a.tail : a.head) + tile * a.dim + col;
        store_v<float, V>(part, acc);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = 0.f;
      began = true;
    }
  }
}

// Number of tiles right behind `tile` that begin with token t: the keys are
// sorted, so they are the first ones, and 32 lanes narrow the range at a time.
__device__ __forceinline__ int64_t tiles_of_run(const GradArgs& a, const uint32_t* key, int64_t tile,
                                                uint32_t t) {
  const int lane = threadIdx.x & 31;
  int64_t lo = 0, hi = a.tiles - 1 - tile;  // the first lo do, none behind the first hi does
  while (lo < hi) {
    const int64_t step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
    const bool on = at <= hi && key[(tile + at) * a.places] == t;
    const int n = __popc(__ballot_sync(0xffffffffu, on));
    const int64_t next = lo + (int64_t)(n + 1) * step - 1;  // the one behind the last hit fails
    lo += (int64_t)n * step;
    hi = next < hi ? next : hi;
  }
  return lo;
}

// One CTA per tile and 32 V columns, and further ones where these outnumber the grid's
// second dimension: if a run begins in the tile and goes on
// behind it, its parts are added in four stretches of tiles, a warp each, and
// the stretches in order.
template <typename TT, int V>
__global__ void __launch_bounds__(kSumThreads) emb_join(const __grid_constant__ GradArgs a) {
  __shared__ float part[kSumThreads / 32][32 * V];
  wait_for_launch_before();
  const int64_t tile = blockIdx.x, p0 = tile * a.places, last = p0 + a.places - 1;
  if (last + 1 >= a.rows) return;
  const uint32_t* key = sorted_key(a);
  const uint32_t t = key[last];
  if (t >= (uint32_t)a.vocab || key[last + 1] != t) return;
  if (p0 > 0 && key[p0] == t && key[p0 - 1] == t) return;  // began earlier
  const int64_t n = tiles_of_run(a, key, tile, t);  // tiles with a head part
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t j0 = tile + 1 + n * warp / 4, j1 = tile + 1 + n * (warp + 1) / 4;
  for (int c0 = blockIdx.y * 32 * V; c0 < a.dim; c0 += gridDim.y * 32 * V) {
    const int col = c0 + lane * V;
    float acc[V] = {};
    if (col < a.dim) {
      if (warp == 0) load_v<float, V>(a.tail + tile * a.dim + col, acc);
      const float* src = a.head + col;
#pragma unroll 8
      for (int64_t j = j0; j < j1; ++j) {
        float v[V];
        load_v<float, V>(src + j * a.dim, v);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += v[e];
      }
#pragma unroll
      for (int e = 0; e < V; ++e) part[warp][lane * V + e] = acc[e];
    }
    __syncthreads();
    if (warp == 0 && col < a.dim) {
#pragma unroll
      for (int w = 1; w < kSumThreads / 32; ++w)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += part[w][lane * V + e];
      store_grad<TT, V>(a, t, col, acc);
    }
    __syncthreads();
  }
}

// Places of a tile: many tiles for short batches, and few parts of a run for
// long ones. (8, 32 and 128 places: 4096 rows of 512 22, 27 and 47 us; 8192 of 1024 51,
// 49 and 70; 32768 of 1024 92, 68 and 78; 131072 of 512 190, 121 and 104; 262144 of 512
// 359, 215 and 187.)
int places_for(int64_t rows) { return rows <= 8192 ? 8 : rows <= 131072 ? 32 : kMaxPlaces; }

struct Layout {
  int64_t tiles, rows_bytes, part_bytes, total;
  int places;
};
Layout layout(int64_t rows, int64_t dim) {
  Layout l;
  l.places = places_for(rows);
  l.tiles = ceil_div(rows, l.places);
  l.rows_bytes = ceil_div(4 * rows, 16) * 16;
  l.part_bytes = ceil_div(4 * l.tiles * dim, 16) * 16;
  l.total = 4 * l.rows_bytes + 2 * l.part_bytes;
  return l;
}

bool vec_ok(const void* p, int64_t ld, magma_dtype_t t, int v) {
  return (reinterpret_cast<uintptr_t>(p) & (std::min<size_t>(16, v * dtype_size(t)) - 1)) == 0 &&
         ld % v == 0;
}

template <typename TD, typename TT, int V>
magma_status_t launch_grad(const GradArgs& a, cudaStream_t cs) {
  // the cluster that sorts, and as many others as there is other work for
  int64_t n = 1;
  while (n < kMaxCluster && n * kSortRows < a.rows) n *= 2;
  const int64_t other = (a.accumulate ? 0 : a.vocab * (int64_t)a.dim) +
                        (a.dpos ? a.seq * a.dim * (a.batch + 1) : 0);
  if (a.rows == 0 && other == 0) return MAGMA_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)n);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = kCountBytes;
  cfg.stream = cs;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)n;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (other > 0) {
    // No more clusters than run at once: a cluster needs its CTAs on one GPC,
    // and the last ones of a second wave would take as long as all of the first.
    int most = 0;
    if (magma_status_t st = cuda_status(
            cudaOccupancyMaxActiveClusters(&most, emb_sort<TD, TT, V>, &cfg), "emb_sort clusters"))
      return st;
    const int64_t more =
        std::min<int64_t>(ceil_div(other, (int64_t)n * kSortThreads * V * 4), most - 1);
    cfg.gridDim = dim3((unsigned)(n * (1 + std::max<int64_t>(more, 0))));
  }
  if (magma_status_t st = cuda_status(cudaLaunchKernelEx(&cfg, emb_sort<TD, TT, V>, a), "emb_sort"))
    return st;
  if (a.tiles == 0) return MAGMA_OK;
  const unsigned cols = (unsigned)ceil_div(a.dim, kSumThreads * V);
  if (magma_status_t st = launch_after(emb_sum<TD, TT, V>, dim3((unsigned)a.tiles, cols),
                                       kSumThreads, 0, cs, "emb_sum", a))
    return st;
  if (a.tiles < 2) return MAGMA_OK;  // no border for a run to cross
  return launch_after(emb_join<TT, V>,
                      dim3((unsigned)(a.tiles - 1),
                           (unsigned)std::min<int64_t>(ceil_div(a.dim, 32 * V), 65535)),
                      kSumThreads, 0, cs, "emb_join", a);
}

template <typename TI, typename TO>
magma_status_t launch_lookup(const int32_t* tokens, const void* table, int64_t ld, const void* pos,
                             void* out, int64_t rows, int64_t seq, int64_t dim, int64_t vocab,
                             float scale, bool vec, cudaStream_t cs) {
  const int64_t blocks = std::min<int64_t>(ceil_div(rows, 4), 0x7FFFFFFF);
  auto* k = vec ? emb_lookup<TI, TO, 8> : emb_lookup<TI, TO, 1>;
  k<<<(unsigned)blocks, 128, 0, cs>>>(tokens, static_cast<const TI*>(table), ld,
                                      static_cast<const TI*>(pos), static_cast<TO*>(out), rows, seq,
                                      (int)dim, vocab, scale, device_error_word());
  return check_launch("emb_lookup");
}

// n rows of dim elements, ld apart.
MemView rows_view(const void* p, int64_t n, int64_t dim, int64_t ld, magma_dtype_t t) {
  const int64_t e = (int64_t)dtype_size(t);
  return {p, dim * e, {n, 1, 1}, {ld * e, 0, 0}};
}

magma_status_t check_sizes(const char* fn, int64_t batch, int64_t seq, int64_t dim, int64_t vocab) {
  MAGMA_REQUIRE(batch >= 0 && seq >= 0 && dim >= 0 && vocab >= 0, "%s: negative size", fn);
  MAGMA_REQUIRE(vocab < 0x7FFFFFFFLL && dim <= (1LL << 22), "%s: vocab or dim too large", fn);
  MAGMA_REQUIRE(batch == 0 || seq <= 0x7FFFFFFFLL / batch, "%s: more than 2^31 - 1 rows", fn);
  MAGMA_REQUIRE(batch > 0 || seq < 0x7FFFFFFFLL, "%s: more than 2^31 - 1 rows", fn);
  return MAGMA_OK;
}

}  // namespace
}  // namespace magma

using namespace magma;

extern "C" {

magma_status_t magma_embedding_scaled_fwd(const int32_t* tokens, const void* table,
                                          int64_t table_ld, const void* pos, void* out,
                                          int64_t batch, int64_t seq, int64_t dim, int64_t vocab,
                                          float scale, magma_dtype_t table_dtype,
                                          magma_dtype_t out_dtype, void* stream) {
  const char* fn = "magma_embedding_scaled_fwd";
  if (magma_status_t st = check_sizes(fn, batch, seq, dim, vocab)) return st;
  MAGMA_REQUIRE(is_float_dtype(table_dtype) && is_float_dtype(out_dtype),
                "%s: dtypes must be F32 or BF16", fn);
  const int64_t rows = batch * seq;
  if (rows == 0 || dim == 0) return MAGMA_OK;
  MAGMA_REQUIRE(vocab > 0, "%s: an empty table", fn);
  MAGMA_REQUIRE(tokens && table && out, "%s: NULL pointer", fn);
  MAGMA_REQUIRE(table_ld >= dim, "%s: table_ld %lld below dim %lld", fn, (long long)table_ld,
                (long long)dim);
  MAGMA_REQUIRE(on_element(tokens, 4) && on_element(table, dtype_size(table_dtype)) &&
                    on_element(pos, dtype_size(table_dtype)) && on_element(out, dtype_size(out_dtype)),
                "%s: an address off its elements", fn);
  const MemView ov = rows_view(out, rows, dim, dim, out_dtype);
  const MemView inputs[] = {rows_view(table, vocab, dim, table_ld, table_dtype),
                            rows_view(pos, seq, dim, dim, table_dtype), {tokens, 4 * rows}};
  for (const MemView& x : inputs)
    MAGMA_REQUIRE(!share_memory(ov, x), "%s: out shares memory with an input", fn);
  const bool vec = vec_ok(table, table_ld, table_dtype, 8) && vec_ok(out, dim, out_dtype, 8) &&
                   (pos == nullptr || vec_ok(pos, dim, table_dtype, 8));
  cudaStream_t cs = (cudaStream_t)stream;
  const bool bi = table_dtype == MAGMA_DTYPE_BF16, bo = out_dtype == MAGMA_DTYPE_BF16;
  auto* run = bi ? (bo ? launch_lookup<__nv_bfloat16, __nv_bfloat16>
                       : launch_lookup<__nv_bfloat16, float>)
                 : (bo ? launch_lookup<float, __nv_bfloat16> : launch_lookup<float, float>);
  return run(tokens, table, table_ld, pos, out, rows, seq, dim, vocab, scale, vec, cs);
}

int64_t magma_embedding_scaled_bwd_workspace_size(int64_t batch, int64_t seq, int64_t dim) {
  if (batch <= 0 || seq <= 0 || dim <= 0 || seq > 0x7FFFFFFFLL / batch) return 0;
  return layout(batch * seq, dim).total;
}

magma_status_t magma_embedding_scaled_bwd(const int32_t* tokens, const void* dout, int64_t dout_ld,
                                          void* dtable, int64_t dtable_ld, float* dpos,
                                          int64_t batch, int64_t seq, int64_t dim, int64_t vocab,
                                          float scale, int64_t padding_idx, int32_t accumulate,
                                          int32_t accumulate_dpos, magma_dtype_t dout_dtype,
                                          magma_dtype_t dtable_dtype, void* workspace,
                                          int64_t workspace_bytes, void* stream) {
  const char* fn = "magma_embedding_scaled_bwd";
  if (magma_status_t st = check_sizes(fn, batch, seq, dim, vocab)) return st;
  MAGMA_REQUIRE(is_float_dtype(dout_dtype) && is_float_dtype(dtable_dtype),
                "%s: dtypes must be F32 or BF16", fn);
  MAGMA_REQUIRE(padding_idx >= -1 && padding_idx < vocab,
                "%s: padding_idx %lld outside the table (-1: none)", fn, (long long)padding_idx);
  if (dim == 0) return MAGMA_OK;
  const int64_t rows = batch * seq;
  MAGMA_REQUIRE(vocab > 0 || rows == 0, "%s: an empty table", fn);
  MAGMA_REQUIRE(vocab == 0 || (dtable && dtable_ld >= dim), "%s: NULL dtable or dtable_ld below dim", fn);
  MAGMA_REQUIRE(rows == 0 || (tokens && dout && dout_ld >= dim),
                "%s: NULL pointer or dout_ld below dim", fn);
  MAGMA_REQUIRE(on_element(tokens, 4) && on_element(dout, dtype_size(dout_dtype)) &&
                    on_element(dtable, dtype_size(dtable_dtype)) && on_element(dpos, 4),
                "%s: an address off its elements", fn);
  const MemView tv = rows_view(dtable, vocab, dim, dtable_ld, dtable_dtype);
  const MemView pv = rows_view(dpos, seq, dim, dim, MAGMA_DTYPE_F32);
  const MemView inputs[] = {rows_view(dout, rows, dim, dout_ld, dout_dtype), {tokens, 4 * rows}};
  for (const MemView& x : inputs)
    MAGMA_REQUIRE(!share_memory(tv, x) && !share_memory(pv, x),
                  "%s: outputs share memory with an input", fn);
  MAGMA_REQUIRE(!share_memory(tv, pv), "%s: dtable and dpos share memory", fn);
  const Layout l = layout(rows, dim);
  MAGMA_REQUIRE(rows == 0 || (workspace && workspace_bytes >= l.total && aligned16(workspace)),
                "%s: a 16-byte aligned workspace of %lld bytes is needed", fn, (long long)l.total);
  cudaStream_t cs = (cudaStream_t)stream;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  GradArgs a{};
  a.tokens = tokens;
  for (int i = 0; i < 2; ++i) {
    a.key[i] = reinterpret_cast<uint32_t*>(ws + i * l.rows_bytes);
    a.row[i] = reinterpret_cast<uint32_t*>(ws + (2 + i) * l.rows_bytes);
  }
  a.head = reinterpret_cast<float*>(ws + 4 * l.rows_bytes);
  a.tail = reinterpret_cast<float*>(ws + 4 * l.rows_bytes + l.part_bytes);
  a.dout = dout;
  a.dout_ld = dout_ld;
  a.dtable = dtable;
  a.dtable_ld = dtable_ld;
  a.dpos = dpos;
  a.rows = rows;
  a.vocab = vocab;
  a.batch = batch;
  a.seq = seq;
  a.padding = padding_idx;
  a.tiles = l.tiles;
  a.dim = (int)dim;
  a.places = l.places;
  // the largest key is `vocab`
  a.passes = vocab < (1 << 8) ? 1 : vocab < (1 << 16) ? 2 : vocab < (1 << 24) ? 3 : 4;
  a.accumulate = accumulate;
  a.accumulate_dpos = accumulate_dpos;
  a.scale = scale;
  a.err = device_error_word();
  // Sixteen-byte accesses of dout where everything is aligned for them, single elements
  // otherwise (32768 rows of 776 BF16 46 us, of 777 76; 16384 F32 rows 40 and 55).
  const int vmax = dout_dtype == MAGMA_DTYPE_BF16 ? 8 : 4;
  const bool vec = vec_ok(dout, dout_ld, dout_dtype, vmax) && dim % 8 == 0 &&
                   aligned16(dtable) && vec_ok(dtable, dtable_ld, dtable_dtype, 8) &&
                   (dpos == nullptr || vec_ok(dpos, dim, MAGMA_DTYPE_F32, vmax));
  const bool bd = dout_dtype == MAGMA_DTYPE_BF16, bt = dtable_dtype == MAGMA_DTYPE_BF16;
  if (vec)
    return bd ? (bt ? launch_grad<__nv_bfloat16, __nv_bfloat16, 8>(a, cs)
                    : launch_grad<__nv_bfloat16, float, 8>(a, cs))
              : (bt ? launch_grad<float, __nv_bfloat16, 4>(a, cs)
                    : launch_grad<float, float, 4>(a, cs));
  return bd ? (bt ? launch_grad<__nv_bfloat16, __nv_bfloat16, 1>(a, cs)
                  : launch_grad<__nv_bfloat16, float, 1>(a, cs))
            : (bt ? launch_grad<float, __nv_bfloat16, 1>(a, cs)
                  : launch_grad<float, float, 1>(a, cs));
}

}  // extern "C"
