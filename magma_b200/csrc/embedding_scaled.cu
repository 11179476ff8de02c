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
//                  end up last.
//  2. emb_sum      a CTA adds the dout rows of P consecutive places of the
//                  sorted order, so that every CTA has the same work however
//                  often a token repeats. A run of equal tokens inside the P
//                  places is stored at once; the part of a run that crosses a
//                  border goes to the workspace. Further CTAs write the zero
//                  rows of tokens that do not occur, and dpos.
//  3. emb_join     adds the parts of each crossing run in order.
// The order of the additions depends on the tokens alone (no atomics on
// floating values), so the result is the same on every run.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"

namespace magma {
namespace {

namespace cg = cooperative_groups;

// ---- lookup --------------------------------------------------------------------
// A warp per row and pass of U vectors a lane, all loads of a pass first. HBM
// bound: the table and position rows are read and the output written once.
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

// ---- sort ----------------------------------------------------------------------
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kDigits = 256;
// A CTA of the cluster takes at least this many rows: below it the exchange of
// the counts costs more than the rows.
constexpr int kSortRows = 2048;

struct SortArgs {
  const int32_t* tokens;
  uint32_t* key[2];  // ping-pong buffers
  uint32_t* row[2];
  int64_t rows;
  int64_t vocab;
  int64_t padding;
  int passes;
  int* err;
};

__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, int64_t i, bool report) {
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
// so equal digits keep their order.
__global__ void __launch_bounds__(kSortThreads, 1) emb_sort(const SortArgs a) {
  extern __shared__ uint32_t counts[];                  // [warp][digit]
  __shared__ uint32_t cta_count[kDigits], scan[kDigits];
  cg::cluster_group cluster = cg::this_cluster();
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
    const uint32_t* kin = a.key[(p + 1) & 1];
    const uint32_t* rin = a.row[(p + 1) & 1];
    uint32_t* kout = a.key[p & 1];
    uint32_t* rout = a.row[p & 1];
    for (int d = lane; d < kDigits; d += 32) mine[d] = 0;
    __syncwarp();
    for (int64_t i = i0 + lane; i < i1; i += 32) {
      const uint32_t k = p == 0 ? sort_key(a, i, true) : kin[i];
      atomicAdd(&mine[(k >> shift) & (kDigits - 1)], 1u);
    }
    __syncthreads();
    // counts[w][d] -> rows of digit d in earlier warps of this CTA
    if (threadIdx.x < kDigits) {
      uint32_t run = 0;
#pragma unroll 8
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
      for (int o = 0; o < nc; ++o) {
        const uint32_t n = cluster.map_shared_rank(cta_count, o)[threadIdx.x];
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
#pragma unroll 8
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
    // the next pass reads what other CTAs of the cluster wrote, and the counts
    // of this one are read by them until here
    __threadfence();
    cluster.sync();
  }
}

// ---- sum -----------------------------------------------------------------------
constexpr int kSumThreads = 128;
constexpr int kMaxPlaces = 128;

struct SumArgs {
  const uint32_t* key;
  const uint32_t* row;
  const void* dout;
  int64_t dout_ld;
  void* dtable;
  int64_t dtable_ld;
  float* head;  // [tile][dim]: the tile's part of a run that began before it
  float* tail;  // [tile][dim]: the tile's part of a run that began in it and goes on
  float* dpos;
  int64_t rows, vocab, batch, seq;
  int64_t tiles, zero_blocks, pos_blocks;
  int dim, places, accumulate, accumulate_dpos;
  float scale;
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

template <typename T, int V>
__device__ __forceinline__ void store_grad(const SumArgs& a, uint32_t token, int col,
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

// First place whose key is at least x.
__device__ __forceinline__ int64_t lower_bound(const uint32_t* key, int64_t n, uint32_t x) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (key[mid] < x) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

constexpr int kZeroRows = 8;  // vocabulary rows of a warp that writes zero rows

template <typename T, int V>
__device__ __forceinline__ void zero_rows(const SumArgs& a, int64_t block) {
  const int lane = threadIdx.x & 31;
  const int64_t v0 = (block * (kSumThreads / 32) + (threadIdx.x >> 5)) * kZeroRows;
  bool absent = false;
  if (lane < kZeroRows && v0 + lane < a.vocab) {
    const uint32_t v = (uint32_t)(v0 + lane);
    const int64_t p = lower_bound(a.key, a.rows, v);
    absent = p == a.rows || a.key[p] != v;
  }
  const uint32_t mask = __ballot_sync(0xffffffffu, absent);
  const float zero[V] = {};
  for (int j = 0; j < kZeroRows; ++j) {
    if (!(mask >> j & 1u)) continue;
    T* dst = static_cast<T*>(a.dtable) + (v0 + j) * a.dtable_ld;
    for (int c = lane * V; c < a.dim; c += 32 * V) store_v<T, V>(dst + c, zero);
  }
}

template <typename TD, int V>
__device__ __forceinline__ void sum_positions(const SumArgs& a, int64_t block) {
  const int64_t nv = a.dim / V;
  const int64_t i = block * kSumThreads + threadIdx.x;
  if (i >= a.seq * nv) return;
  const int64_t s = i / nv;
  const int col = (int)(i % nv) * V;
  float acc[V] = {};
  const TD* src = static_cast<const TD*>(a.dout) + s * a.dout_ld + col;
  float* dst = a.dpos + s * a.dim + col;
#pragma unroll 4
  for (int64_t b = 0; b < a.batch; ++b) {
    float v[V];
    load_v<TD, V>(src + b * a.seq * a.dout_ld, v);
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] += v[e];
  }
#pragma unroll
  for (int e = 0; e < V; ++e) dst[e] = a.accumulate_dpos ? dst[e] + acc[e] : acc[e];
}

// TD: dout, TT: dtable. The dout rows of eight places are in flight at a time.
template <typename TD, typename TT, int V>
__global__ void __launch_bounds__(kSumThreads) emb_sum(const SumArgs a) {
  if ((int64_t)blockIdx.x >= a.tiles) {
    const int64_t b = (int64_t)blockIdx.x - a.tiles;
    if (blockIdx.y != 0) return;
    if (b < a.zero_blocks) zero_rows<TT, V>(a, b);
    else sum_positions<TD, V>(a, b - a.zero_blocks);
    return;
  }
  __shared__ uint32_t key[kMaxPlaces + 2], row[kMaxPlaces];
  const int64_t tile = blockIdx.x, p0 = tile * a.places;
  const int n = (int)(a.rows - p0 < a.places ? a.rows - p0 : a.places);
  // key[0]: the place before the tile, key[n + 1]: the place behind it
  for (int i = threadIdx.x; i < n + 2; i += kSumThreads) {
    const int64_t p = p0 + i - 1;
    key[i] = p >= 0 && p < a.rows ? a.key[p] : 0xFFFFFFFFu;
    if (i >= 1 && i <= n) row[i - 1] = a.row[p];
  }
  __syncthreads();
  const int col = (blockIdx.y * kSumThreads + threadIdx.x) * V;
  if (col >= a.dim) return;
  const TD* src = static_cast<const TD*>(a.dout) + col;
  float acc[V] = {};
  bool began = key[0] != key[1];  // the current run begins in this tile
  constexpr int kAhead = 8;
  for (int i0 = 0; i0 < n; i0 += kAhead) {
    float v[kAhead][V];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (i0 + u < n && key[i0 + u + 1] < (uint32_t)a.vocab)
        load_v<TD, V>(src + (int64_t)row[i0 + u] * a.dout_ld, v[u]);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u;
      if (i >= n) break;
      const uint32_t t = key[i + 1];
      if (t >= (uint32_t)a.vocab) return;  // padding and bad tokens are last
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += v[u][e];
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

// One CTA per tile: if a run begins in the tile and goes on behind it, adds its
// parts in order.
template <typename TT, int V>
__global__ void __launch_bounds__(kSumThreads) emb_join(const SumArgs a) {
  const int64_t tile = blockIdx.x, p0 = tile * a.places, last = p0 + a.places - 1;
  if (last + 1 >= a.rows) return;
  const uint32_t t = a.key[last];
  if (t >= (uint32_t)a.vocab || a.key[last + 1] != t) return;
  if (p0 > 0 && a.key[p0] == t && a.key[p0 - 1] == t) return;  // began earlier
  const int64_t end = lower_bound(a.key, a.rows, t + 1);       // behind the run
  const int64_t last_tile = (end - 1) / a.places;
  const int col = (blockIdx.y * kSumThreads + threadIdx.x) * V;
  if (col >= a.dim) return;
  float acc[V];
  load_v<float, V>(a.tail + tile * a.dim + col, acc);
#pragma unroll 8
  for (int64_t j = tile + 1; j <= last_tile; ++j) {
    float v[V];
    load_v<float, V>(a.head + j * a.dim + col, v);
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] += v[e];
  }
  store_grad<TT, V>(a, t, col, acc);
}

// Places of a tile: many tiles for short batches, and few parts of a run for
// long ones.
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
magma_status_t launch_sum(const SumArgs& a, cudaStream_t cs) {
  const unsigned cols = (unsigned)ceil_div(a.dim, kSumThreads * V);
  const int64_t blocks = a.tiles + a.zero_blocks + a.pos_blocks;
  if (blocks > 0x7FFFFFFFLL) return fail(MAGMA_INVALID_ARGUMENT, "magma_embedding_scaled_bwd: too large");
  emb_sum<TD, TT, V><<<dim3((unsigned)blocks, cols), kSumThreads, 0, cs>>>(a);
  if (magma_status_t st = check_launch("emb_sum")) return st;
  if (a.tiles < 2) return MAGMA_OK;  // no border for a run to cross
  emb_join<TT, V><<<dim3((unsigned)(a.tiles - 1), cols), kSumThreads, 0, cs>>>(a);
  return check_launch("emb_join");
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

magma_status_t check_sizes(const char* fn, int64_t batch, int64_t seq, int64_t dim, int64_t vocab) {
  MAGMA_REQUIRE(batch >= 0 && seq >= 0 && dim >= 0 && vocab >= 0, "%s: negative size", fn);
  MAGMA_REQUIRE(vocab < 0x7FFFFFFFLL && dim <= (1LL << 22), "%s: vocab or dim too large", fn);
  MAGMA_REQUIRE(batch == 0 || seq <= 0x7FFFFFFFLL / batch, "%s: more than 2^31 - 1 rows", fn);
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
  const Layout l = layout(rows, dim);
  MAGMA_REQUIRE(rows == 0 || (workspace && workspace_bytes >= l.total && aligned16(workspace)),
                "%s: a 16-byte aligned workspace of %lld bytes is needed", fn, (long long)l.total);
  cudaStream_t cs = (cudaStream_t)stream;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  SortArgs s{};
  s.tokens = tokens;
  for (int i = 0; i < 2; ++i) {
    s.key[i] = reinterpret_cast<uint32_t*>(ws + i * l.rows_bytes);
    s.row[i] = reinterpret_cast<uint32_t*>(ws + (2 + i) * l.rows_bytes);
  }
  s.rows = rows;
  s.vocab = vocab;
  s.padding = padding_idx;
  s.passes = vocab < (1 << 8) ? 1 : vocab < (1 << 16) ? 2 : vocab < (1 << 24) ? 3 : 4;
  s.err = device_error_word();
  if (rows > 0) {
    int64_t n = 1;
    while (n < kMaxCluster && n * kSortRows < rows) n *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n);
    cfg.blockDim = dim3(kSortThreads);
    cfg.dynamicSmemBytes = kSortWarps * kDigits * 4;
    cfg.stream = cs;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)n;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (magma_status_t st = cuda_status(cudaLaunchKernelEx(&cfg, emb_sort, s), "emb_sort"))
      return st;
  }
  SumArgs a{};
  a.key = s.key[(s.passes - 1) & 1];
  a.row = s.row[(s.passes - 1) & 1];
  a.dout = dout;
  a.dout_ld = dout_ld;
  a.dtable = dtable;
  a.dtable_ld = dtable_ld;
  a.head = reinterpret_cast<float*>(ws + 4 * l.rows_bytes);
  a.tail = reinterpret_cast<float*>(ws + 4 * l.rows_bytes + l.part_bytes);
  a.dpos = dpos;
  a.rows = rows;
  a.vocab = vocab;
  a.batch = batch;
  a.seq = seq;
  a.dim = (int)dim;
  a.places = l.places;
  a.tiles = l.tiles;
  a.accumulate = accumulate;
  a.accumulate_dpos = accumulate_dpos;
  a.scale = scale;
  // Sixteen-byte accesses of dout where everything is aligned for them.
  const int vmax = dout_dtype == MAGMA_DTYPE_BF16 ? 8 : 4;
  const bool vec = vec_ok(dout, dout_ld, dout_dtype, vmax) && dim % vmax == 0 &&
                   vec_ok(dtable, dtable_ld, dtable_dtype, vmax) &&
                   (dpos == nullptr || vec_ok(dpos, dim, MAGMA_DTYPE_F32, vmax));
  const int v = vec ? vmax : 1;
  a.zero_blocks = accumulate ? 0 : ceil_div(vocab, kZeroRows * (kSumThreads / 32));
  a.pos_blocks = dpos == nullptr ? 0 : ceil_div(seq * (dim / v), kSumThreads);
  if (a.tiles + a.zero_blocks + a.pos_blocks == 0) return MAGMA_OK;
  const bool bd = dout_dtype == MAGMA_DTYPE_BF16, bt = dtable_dtype == MAGMA_DTYPE_BF16;
  if (vec)
    return bd ? (bt ? launch_sum<__nv_bfloat16, __nv_bfloat16, 8>(a, cs)
                    : launch_sum<__nv_bfloat16, float, 8>(a, cs))
              : (bt ? launch_sum<float, __nv_bfloat16, 4>(a, cs)
                    : launch_sum<float, float, 4>(a, cs));
  return bd ? (bt ? launch_sum<__nv_bfloat16, __nv_bfloat16, 1>(a, cs)
                  : launch_sum<__nv_bfloat16, float, 1>(a, cs))
            : (bt ? launch_sum<float, __nv_bfloat16, 1>(a, cs)
                  : launch_sum<float, float, 1>(a, cs));
}

}  // extern "C"
