// Attention of a few queries over long sources: one query per sequence (a
// decoding step) or a handful, times the heads that share a key head.
//
// The work is one read of K and V (4 flops per byte and query row), so the
// source is cut into chunks, a CTA takes one chunk of one key head with all
// query rows that read it (row = shared head * q_len + query), and the parts
// are joined by their log-sum-exp: by the cluster that the chunks of a short source
// form, through distributed shared memory, or by cross_join_parts. Keys from the length on
// are filled with zeros: what lies behind a length is never read.
// Bound by HBM for many sources (BF16, 64 x 32 heads over 8 of 128, up to 4096 keys,
// 678 MB: 107 us, 6.3 TB/s, and 6 us for the join), by a launch and two trips to
// memory for one (16 heads of 64, 777 keys, 3.2 MB: 7 us, one launch).
//
//   cross_step_bf16  warp-level MMA (m16n8k16): WM x (4 / WM) warps over rows
//                    and keys, each with its own running maximum and sum. The
//                    16-row tile holds one query of up to 16 heads; the tcgen05
//                    tile of 128 rows would be empty, and the products are not
//                    what bounds this. K and V tiles come through a cp.async ring.
//   cross_step_f32   FMA pipe: scores by key, sums by column, four warps over
//                    the keys.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

#include "cross_attention.cuh"
#include "sm100.cuh"

namespace magma {
namespace {

using namespace sm100;
namespace cg = cooperative_groups;

constexpr int kThreads = 128;
constexpr int kMaxCluster = 8;
constexpr int kKeys = 64;  // keys of a BF16 tile
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct StepArgs {
  CrossGeom g;
  int rows;             // shared heads * q_len
  int groups, each;     // CTAs that share a chunk's rows, rows of one of them
  int n_chunk;          // chunks of the longest source
  int64_t chunk;        // keys of a chunk, a multiple of the tile
  int cluster;          // the chunks of a source are a cluster, which joins them itself
  void* o;
  float* lse;
  float* part;          // [chunk][b][h][q][hd], of several chunks that are no cluster
  float* part_lse;      // [chunk][b][h][q], natural logarithm
};

// One CTA's chunk: sequence, key head, keys [k0, k1), first of its query rows.
struct Chunk {
  int64_t b, kvh, k0, k1;
  int index, r0;
};
__device__ __forceinline__ Chunk chunk_of(const StepArgs& a) {
  Chunk c;
  int64_t i = blockIdx.x;
  c.index = (int)(i % a.n_chunk);
  i /= a.n_chunk;
  c.r0 = (int)(i % a.groups) * a.each;
  i /= a.groups;
  c.kvh = i % a.g.kv_heads;
  c.b = i / a.g.kv_heads;
  const int64_t len = cross_len(a.g, c.b);
  c.k0 = c.index * a.chunk < len ? c.index * a.chunk : len;
  c.k1 = len - c.k0 < a.chunk ? len : c.k0 + a.chunk;
  return c;
}

// Index of packed row r in a [b][h][q] array, and its head and query.
__device__ __forceinline__ int64_t row_at(const CrossGeom& g, const Chunk& c, int r, int64_t* h,
                                          int64_t* q) {
  *h = c.kvh * g.group + r / (int)g.q_len;
  *q = r % (int)g.q_len;
  return (c.b * g.heads + *h) * g.q_len + *q;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(on ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

// Stores a row's result: the output itself, or a chunk's normalised part.
template <typename T>
__device__ __forceinline__ void store_part(const StepArgs& a, const Chunk& c, int r, int col,
                                           const float (&v)[4], float lse) {
  int64_t h, q;
  const int64_t at = row_at(a.g, c, r, &h, &q);
  const int64_t rows = a.g.batch * a.g.heads * a.g.q_len;
  if (a.part != nullptr) {
    store4(a.part + (c.index * rows + at) * a.g.hd + col, v);
    if (col == 0) a.part_lse[c.index * rows + at] = lse;
  } else {
    store4(static_cast<T*>(a.o) + c.b * a.g.os[0] + h * a.g.os[1] + q * a.g.os[2] + col, v);
    if (col == 0 && a.lse != nullptr) a.lse[at] = lse;
  }
}

// exp in the base that a kernel keeps its maxima in, and a maximum as a natural
// logarithm.
template <bool LOG2> __device__ __forceinline__ float exp_of(float x) {
  if constexpr (LOG2) return ex2_approx(x);
  else return expf(x);
}
template <bool LOG2> __device__ __forceinline__ float ln_of(float x) { return LOG2 ? x * kLn2 : x; }

// The CTA's sums over its warps, and those of the cluster's CTAs. so: [warp][R][P]
// sums, relative to the maximum in sml[warp * R + row]; WN warps share a row of
// ROWS. A row's sum over the warps is put in the place of its first warp's, where
// the other CTAs read it. fin: [ROWS].
template <typename T, bool LOG2, int ROWS, int R, int WN, int HD, int P>
__device__ __forceinline__ void finish(const StepArgs& a, const Chunk& c, float* so,
                                       const float2* sml, float2* fin) {
  constexpr int kVec = HD / 4;
  const int tid = threadIdx.x;
  for (int i = tid; i < ROWS * kVec; i += kThreads) {
    const int r = i / kVec, col = i % kVec * 4;
    if (c.r0 + r >= a.rows || col >= a.g.hd) continue;
    const int w0 = r / R * WN, rr = r % R;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < WN; ++w) mm = fmaxf(mm, sml[(w0 + w) * R + rr].x);
    float total = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WN; ++w) {
      const float2 ml = sml[(w0 + w) * R + rr];
      const float f = mm == -INFINITY ? 0.f : exp_of<LOG2>(ml.x - mm);
      total += f * ml.y;
      float x[4];
      load4(so + ((w0 + w) * R + rr) * P + col, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(f, x[e], o[e]);
    }
    if (a.cluster) {
      store4(so + (w0 * R + rr) * P + col, o);
      if (col == 0) fin[r] = make_float2(mm, total);
      continue;
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= inv;
    store_part<T>(a, c, c.r0 + r, col, o, total == 0.f ? -INFINITY : ln_of<LOG2>(mm) + logf(total));
  }
  if (!a.cluster) return;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int i = c.index * kThreads + tid; i < ROWS * kVec; i += a.n_chunk * kThreads) {
    const int r = i / kVec, col = i % kVec * 4;
    if (c.r0 + r >= a.rows || col >= a.g.hd) continue;
    const int at = (r / R * WN * R + r % R) * P + col;
    float2 ml[kMaxCluster];
    float mm = -INFINITY;
#pragma unroll
    for (int k = 0; k < kMaxCluster; ++k) {
      if (k >= a.n_chunk) continue;
      ml[k] = cluster.map_shared_rank(fin, k)[r];
      mm = fmaxf(mm, ml[k].x);
    }
    float total = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kMaxCluster; ++k) {
      if (k >= a.n_chunk) continue;
      const float f = mm == -INFINITY ? 0.f : exp_of<LOG2>(ml[k].x - mm);
      total += f * ml[k].y;
      const float4 x = *reinterpret_cast<const float4*>(cluster.map_shared_rank(so, k) + at);
      o[0] = fmaf(f, x.x, o[0]);
      o[1] = fmaf(f, x.y, o[1]);
      o[2] = fmaf(f, x.z, o[2]);
      o[3] = fmaf(f, x.w, o[3]);
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= inv;
    store_part<T>(a, c, c.r0 + r, col, o, total == 0.f ? -INFINITY : ln_of<LOG2>(mm) + logf(total));
  }
  cluster.sync();  // the others have read this CTA's sums
}

// ---------------------------------------------------------------- BF16
template <int HD>
struct Bf {
  static constexpr int kStages = HD == 64 ? 3 : 2;
  static constexpr int kChunks = HD / 8;            // 16-byte pieces of a row
  static constexpr int kTile = kKeys * HD * 2;
  static constexpr int kSmem = kStages * 2 * kTile;
  static constexpr int kJoin = 4 * 16 * (HD + 4) * 4;  // the warps' sums at the end
  static_assert(kJoin + 4 * 16 * 8 <= kSmem, "shared memory");
};

template <int HD, int WM>
__global__ void __launch_bounds__(kThreads)
cross_step_bf16(const void* __restrict__ qv, const void* __restrict__ kv,
                const void* __restrict__ vv, const __grid_constant__ StepArgs a) {
  const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(qv);
  const __nv_bfloat16* k = static_cast<const __nv_bfloat16*>(kv);
  const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(vv);
  using F = Bf<HD>;
  constexpr int WN = 4 / WM;         // warps over the keys of a tile
  constexpr int KW = kKeys / WN;     // keys of a warp
  constexpr int NT = KW / 8;         // its 8-key tiles
  constexpr int DT = HD / 8;         // 8-column tiles of the output
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ float2 fin[WM * 16];
  const uint32_t base = smem_u32(sm);
  const CrossGeom& g = a.g;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wm = warp / WN, wn = warp % WN;
  const Chunk c = chunk_of(a);
  const int tiles = (int)((c.k1 - c.k0 + kKeys - 1) / kKeys);

  // tile loads: 16 bytes a thread, a row's pieces side by side
  const int piece = tid % F::kChunks, row0 = tid / F::kChunks;
  constexpr int kRowStep = kThreads / F::kChunks;
  const bool piece_on = piece * 8 < g.hd;
  const __nv_bfloat16* kh = k + c.b * g.ks[0] + c.kvh * g.ks[1] + (piece_on ? piece * 8 : 0);
  const __nv_bfloat16* vh = v + c.b * g.vs[0] + c.kvh * g.vs[1] + (piece_on ? piece * 8 : 0);
  auto load = [&](int j) {
    const uint32_t dst = base + (j % F::kStages) * 2 * F::kTile;
    const int64_t kj = c.k0 + (int64_t)j * kKeys;
#pragma unroll
    for (int i = 0; i < kKeys / kRowStep; ++i) {
      const int r = row0 + i * kRowStep;
      const bool on = piece_on && kj + r < c.k1;
      const int64_t at = on ? kj + r : c.k0;
      const uint32_t o = r * HD * 2 + ((piece ^ (r & 7)) << 4);
      cp_async16(dst + o, kh + at * g.ks[2], on);
      cp_async16(dst + F::kTile + o, vh + at * g.vs[2], on);
    }
  };
#pragma unroll
  for (int j = 0; j < F::kStages - 1; ++j) {
    if (j < tiles) load(j);
    cp_commit();
  }

  // Q fragments: rows lane / 4 and + 8 of the warp's 16
  uint32_t qf[HD / 16][4];
  {
    const __nv_bfloat16* qp[2];
    bool on[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = wm * 16 + (lane >> 2) + 8 * i;
      on[i] = r < a.rows;
      int64_t h, qi;
      row_at(g, c, on[i] ? r : 0, &h, &qi);
      qp[i] = q + c.b * g.qs[0] + h * g.qs[1] + qi * g.qs[2];
    }
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int col = kk * 16 + (lane & 3) * 2 + (e >> 1) * 8;
        qf[kk][e] = on[e & 1] && col < g.hd
                        ? *reinterpret_cast<const uint32_t*>(qp[e & 1] + col) : 0u;
      }
  }
  const float sl2 = g.scale * kLog2e;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float acc[DT][4];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;

  for (int j = 0; j < tiles; ++j) {
    cp_wait<F::kStages - 2>();
    __syncthreads();
    if (j + F::kStages - 1 < tiles) load(j + F::kStages - 1);
    cp_commit();
    const uint32_t sk = base + (j % F::kStages) * 2 * F::kTile, sv = sk + F::kTile;
    const int left = (int)(c.k1 - c.k0 - (int64_t)j * kKeys) - wn * KW;  // keys of this warp
    if (left <= 0) continue;
    float s[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
      for (int p = 0; p < NT / 2; ++p) {
        // keys 16 p .. + 15, columns 16 kk .. + 15: lanes 0-7, 8-15 the first eight
        // keys' two halves, 16-31 the other eight keys'
        const int r = wn * KW + p * 16 + (lane & 7) + ((lane >> 4) << 3);
        const int ch = kk * 2 + ((lane >> 3) & 1);
        uint32_t b[4];
        ldmatrix4(sk + r * HD * 2 + ((ch ^ (r & 7)) << 4), b);
        mma16816(s[2 * p], qf[kk], b[0], b[1]);
        mma16816(s[2 * p + 1], qf[kk], b[2], b[3]);
      }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = i * 8 + (lane & 3) * 2 + (e & 1);
        s[i][e] = key < left ? s[i][e] * sl2 : -INFINITY;
        mx[e >> 1] = fmaxf(mx[e >> 1], s[i][e]);
      }
    float alpha[2], ref[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
      const float mn = fmaxf(m[i], mx[i]);
      ref[i] = mn == -INFINITY ? 0.f : mn;
      alpha[i] = ex2_approx(m[i] - ref[i]);
      m[i] = mn;
      l[i] *= alpha[i];
    }
    uint32_t pf[NT / 2][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[e] = ex2_approx(s[i][e] - ref[e >> 1]);
        l[e >> 1] += p[e];
      }
      // P goes into the second product as BF16, as the operands are: the output's error
      // is 1.2 to 1.3 times that of its own rounding. (With what the rounding left as a
      // second term 1.0 times, in 1 to 7% more time for one query a sequence and 16 to
      // 19% more for 40 to 64 rows a key head.)
      pf[i >> 1][(i & 1) * 2] = pack_bf16(p[0], p[1]);
      pf[i >> 1][(i & 1) * 2 + 1] = pack_bf16(p[2], p[3]);
    }
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] *= alpha[e >> 1];
#pragma unroll
    for (int p = 0; p < NT / 2; ++p)
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) {
        const int r = wn * KW + p * 16 + (lane & 15);
        const int ch = d * 2 + (lane >> 4);
        uint32_t b[4];
        ldmatrix4_t(sv + r * HD * 2 + ((ch ^ (r & 7)) << 4), b);
        mma16816(acc[2 * d], pf[p], b[0], b[1]);
        mma16816(acc[2 * d + 1], pf[p], b[2], b[3]);
      }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
  }
  // the warps' sums meet in shared memory: [warp][16][HD + 4], then (m, l)
  cp_wait<0>();
  __syncthreads();
  float* so = reinterpret_cast<float*>(sm);
  float2* sml = reinterpret_cast<float2*>(sm + F::kJoin);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = (lane >> 2) + 8 * i;
    float* dst = so + (warp * 16 + r) * (HD + 4) + (lane & 3) * 2;
#pragma unroll
    for (int d = 0; d < DT; ++d)
      *reinterpret_cast<float2*>(dst + d * 8) = make_float2(acc[d][2 * i], acc[d][2 * i + 1]);
    if ((lane & 3) == 0) sml[warp * 16 + r] = make_float2(m[i], l[i]);
  }
  __syncthreads();
  finish<__nv_bfloat16, true, WM * 16, 16, WN, HD, HD + 4>(a, c, so, sml, fin);
}

// ----------------------------------------------------------------- F32
// A warp takes groups of eight keys straight from memory into registers (no
// value of K or V is used by two warps) and has its own maximum and sum, so the
// warps run free of one another. Scores: lane = (key, every fourth 16-byte piece
// of d); the next group's K is on its way under the sums, its V under the next
// scores. Sums: lane = four columns, of every key (head size 128) or of every
// second one (64).
constexpr int kF32Keys = 32;  // keys of the four warps' groups

template <int HD, int RT>
__global__ void __launch_bounds__(kThreads, RT == 8 ? 3 : HD == 128 ? 4 : 5)
cross_step_f32(const void* __restrict__ qv, const void* __restrict__ kv,
               const void* __restrict__ vv, const __grid_constant__ StepArgs a) {
  const float* q = static_cast<const float*>(qv);
  const float* k = static_cast<const float*>(kv);
  const float* v = static_cast<const float*>(vv);
  constexpr int kPieces = HD / 16;         // of a lane's share of a K row
  constexpr int kHalves = 128 / HD;        // keys that a V load covers
  constexpr int kLoads = 8 / kHalves;      // V loads of a group
  constexpr int kVec = HD / 4;
  __shared__ __align__(16) float sh[4 * RT * HD];  // q, at the end the warps' sums
  __shared__ float2 sml[4 * RT], fin[RT];
  const CrossGeom& g = a.g;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kk = lane >> 2, part = lane & 3;
  const int vk = lane / kVec, vcol = lane % kVec * 4;  // key of a pair, first column
  const Chunk c = chunk_of(a);
  const int keys = (int)(c.k1 - c.k0), groups = (keys + 7) / 8;
  const float* kh = k + c.b * g.ks[0] + c.kvh * g.ks[1] + c.k0 * g.ks[2];
  const float* vh = v + c.b * g.vs[0] + c.kvh * g.vs[1] + c.k0 * g.vs[2];
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  float4 kx[kPieces], vx[kLoads];
  auto load_k = [&](int grp) {
    const int key = grp * 8 + kk;
    const float* src = kh + key * g.ks[2];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int d = (part + 4 * i) * 4;
      kx[i] = key < keys && d < g.hd ? __ldg(reinterpret_cast<const float4*>(src + d)) : zero;
    }
  };
  auto load_v = [&](int grp) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int key = grp * 8 + i * kHalves + vk;
      vx[i] = key < keys && vcol < g.hd
                  ? __ldg(reinterpret_cast<const float4*>(vh + key * g.vs[2] + vcol)) : zero;
    }
  };
  if (warp < groups) {
    load_k(warp);
    load_v(warp);
  }
  for (int i = tid; i < RT * HD; i += kThreads) {
    const int r = i / HD, col = i % HD;
    float x = 0.f;
    if (c.r0 + r < a.rows && col < g.hd) {
      int64_t h, qi;
      row_at(g, c, c.r0 + r, &h, &qi);
      x = q[c.b * g.qs[0] + h * g.qs[1] + qi * g.qs[2] + col];
    }
    sh[i] = x;
  }
  __syncthreads();
  float m[RT], l[RT], acc[RT][4];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[r][e] = 0.f;
  }
  for (int grp = warp; grp < groups; grp += 4) {
    const int left = keys - grp * 8;
    float s[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) s[r] = 0.f;
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const float4 y = *reinterpret_cast<const float4*>(sh + r * HD + (part + 4 * i) * 4);
        s[r] = fmaf(kx[i].x, y.x, s[r]);
        s[r] = fmaf(kx[i].y, y.y, s[r]);
        s[r] = fmaf(kx[i].z, y.z, s[r]);
        s[r] = fmaf(kx[i].w, y.w, s[r]);
      }
    if (grp + 4 < groups) load_k(grp + 4);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      s[r] += __shfl_xor_sync(0xffffffffu, s[r], 1);
      s[r] += __shfl_xor_sync(0xffffffffu, s[r], 2);
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float x = kk < left ? s[r] * g.scale : -INFINITY;
      float mx = x;
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float mn = fmaxf(m[r], mx);
      const float ref = mn == -INFINITY ? 0.f : mn;
      const float alpha = expf(m[r] - ref);
      m[r] = mn;
      s[r] = expf(x - ref);
      l[r] = l[r] * alpha + s[r];  // the lane's key; a key's four lanes hold the same
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[r][e] *= alpha;
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const float p = __shfl_sync(0xffffffffu, s[r], (i * kHalves + vk) * 4);
        acc[r][0] = fmaf(p, vx[i].x, acc[r][0]);
        acc[r][1] = fmaf(p, vx[i].y, acc[r][1]);
        acc[r][2] = fmaf(p, vx[i].z, acc[r][2]);
        acc[r][3] = fmaf(p, vx[i].w, acc[r][3]);
      }
    if (grp + 4 < groups) load_v(grp + 4);
  }
  __syncthreads();  // q has been used
#pragma unroll
  for (int r = 0; r < RT; ++r) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (kHalves == 2) acc[r][e] += __shfl_xor_sync(0xffffffffu, acc[r][e], 16);
    if (vk == 0) store4(sh + (warp * RT + r) * HD + vcol, acc[r]);
    if (lane == 0) sml[warp * RT + r] = make_float2(m[r], l[r]);
  }
  __syncthreads();
  finish<float, false, RT, RT, 4, HD, HD>(a, c, sh, sml, fin);
}

// ---------------------------------------------------------------- host side
bool step_aligned(const void* p, const int64_t (&st)[3], int64_t per16) {
  return aligned16(p) && st[0] % per16 == 0 && st[1] % per16 == 0 && st[2] % per16 == 0;
}

int64_t tile_keys(magma_dtype_t dtype) { return dtype == MAGMA_DTYPE_F32 ? kF32Keys : kKeys; }

// Rows of a CTA: F32 rows beyond eight go to further CTAs, which read the chunk
// again out of L2 (16 rows in one CTA took half again as long: a thread's sums
// leave no room for enough CTAs to cover the loads).
int rows_each(const CrossGeom& g, magma_dtype_t dtype) {
  const int64_t rows = (int64_t)g.group * g.q_len;
  return dtype == MAGMA_DTYPE_F32 ? (rows <= 4 ? 4 : 8) : (int)rows;
}

// Keys of a chunk: sixteen CTAs per SM, so that lengths that differ even out, but
// chunks below 256 keys only where there are not four CTAs per SM, which is what
// runs at once: each chunk costs a part and its share of the join. (F32, 4 x 32
// heads over 8, 4000 keys: six CTAs per SM 39 us, four 31 us, two 32 us.)
int64_t chunk_keys(const CrossGeom& g, magma_dtype_t dtype) {
  const int64_t tile = tile_keys(dtype);
  const int64_t heads =
      g.batch * g.kv_heads * ceil_div((int64_t)g.group * g.q_len, rows_each(g, dtype));
  const int64_t many = ceil_div(g.kv_len * heads, 16LL * num_sms());
  const int64_t few = ceil_div(g.kv_len * heads, 4LL * num_sms());
  const int64_t keys = std::max(many, std::min<int64_t>(256, few));
  return ceil_div(keys, tile) * tile;
}

// Whether the chunks of a source are the CTAs of a cluster: eight of them for heads
// that do not fill the GPU, while a CTA's chunk stays short. (BF16,
// head size 64: 8 heads, 1000 keys 5.6 us in clusters, 7.0 us with the join; 4 x 8
// heads, 2000 keys 7.6 and 9.3 us; F32, 4 x 32 heads over 8, 4000 keys 39 and 31 us.)
bool use_cluster(const CrossGeom& g, magma_dtype_t dtype) {
  const int64_t heads =
      g.batch * g.kv_heads * ceil_div((int64_t)g.group * g.q_len, rows_each(g, dtype));
  return heads * kMaxCluster <= 6LL * num_sms() && g.kv_len <= (dtype == MAGMA_DTYPE_F32 ? 2048 : 4096);
}

template <typename K>
magma_status_t launch_step(K kernel, const void* q, const void* k, const void* v, const StepArgs& a,
                           unsigned ctas, int smem, cudaStream_t s, const char* what) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.cluster ? (unsigned)a.n_chunk : 1u;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.cluster ? 1 : 0;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, q, k, v, a), what);
}

template <int HD, int WM>
magma_status_t launch_bf16(const void* q, const void* k, const void* v, const StepArgs& a,
                           unsigned ctas, cudaStream_t s) {
  const int smem = Bf<HD>::kSmem;
  if (magma_status_t st = cross_smem<cross_step_bf16<HD, WM>>(smem)) return st;
  return launch_step(cross_step_bf16<HD, WM>, q, k, v, a, ctas, smem, s, "cross_step_bf16");
}

template <int HD, int RT>
magma_status_t launch_f32(const void* q, const void* k, const void* v, const StepArgs& a,
                          unsigned ctas, cudaStream_t s) {
  return launch_step(cross_step_f32<HD, RT>, q, k, v, a, ctas, 0, s, "cross_step_f32");
}

}  // namespace

bool cross_step_supported(const void* q, const void* k, const void* v, const void* o,
                          const CrossGeom& g, magma_dtype_t dtype) {
  const int64_t per16 = dtype == MAGMA_DTYPE_F32 ? 4 : 8;
  return cross_step_rows(g, dtype) && step_aligned(q, g.qs, per16) && step_aligned(k, g.ks, per16) &&
         step_aligned(v, g.vs, per16) && step_aligned(o, g.os, per16);
}

// One to a few rows read K and V once here and leave the tensor cores' or FMA tiles
// nearly empty there (BF16, 16 x 64 heads over 8 of 128, 2000 keys, 8 rows a key head: 35
// and 123 us; 2 x 32 over 4, 4000 keys, 64 rows: 21 and 24; F32, 8 x 8 heads of 64, 1000
// keys, 4 rows: 14 and 32; 8 rows 30 and 31). The limits are as far as the kernels' tiles
// go without giving up that for single requests; batches with many rows a key head do
// better there (BF16, 8 x 8 heads, 1000 keys, 16 rows 10 and 14 us, 32 rows 17 and 15, 64
// rows 20 and 17; 32 x 8 heads of 128, 2000 keys, 64 rows 142 and 59; F32, 16 rows 38 and 31).
bool cross_step_rows(const CrossGeom& g, magma_dtype_t dtype) {
  const int64_t rows = (int64_t)g.group * g.q_len;
  const bool f32 = dtype == MAGMA_DTYPE_F32;
  return rows >= 1 && rows <= (f32 ? 16 : 64) && g.kv_len > 0 && g.hd % (f32 ? 4 : 8) == 0 &&
         g.batch * g.kv_heads * 64 * ceil_div(g.kv_len, 32) < (1LL << 31);
}

size_t cross_step_workspace(const CrossGeom& g, magma_dtype_t dtype) {
  if (use_cluster(g, dtype)) return 0;
  const int64_t n = ceil_div(g.kv_len, chunk_keys(g, dtype));
  return n <= 1 ? 0 : (size_t)n * g.batch * g.heads * g.q_len * (g.hd + 1) * sizeof(float);
}

magma_status_t cross_step_run(const void* q, const void* k, const void* v, void* o, float* lse,
                              const CrossGeom& g, magma_dtype_t dtype, void* workspace,
                              size_t workspace_bytes, cudaStream_t s) {
  StepArgs a{};
  a.g = g;
  a.rows = (int)(g.group * g.q_len);
  a.each = rows_each(g, dtype);
  a.groups = (int)ceil_div(a.rows, a.each);
  a.o = o;
  a.lse = lse;
  const int64_t tile = tile_keys(dtype);
  const int64_t rows = g.batch * g.heads * g.q_len;
  const size_t each = (size_t)rows * (g.hd + 1) * sizeof(float);
  a.cluster = use_cluster(g, dtype) ? 1 : 0;
  a.chunk = a.cluster ? ceil_div(g.kv_len, kMaxCluster * tile) * tile : chunk_keys(g, dtype);
  const int64_t room = workspace && aligned16(workspace) ? (int64_t)(workspace_bytes / each) : 0;
  if (!a.cluster && ceil_div(g.kv_len, a.chunk) > std::max<int64_t>(1, room))
    a.chunk = ceil_div(g.kv_len, std::max<int64_t>(1, room) * tile) * tile;
  a.n_chunk = (int)ceil_div(g.kv_len, a.chunk);
  if (a.n_chunk == 1) a.cluster = 0;
  if (a.n_chunk > 1 && !a.cluster) {
    a.part = static_cast<float*>(workspace);
    a.part_lse = a.part + (size_t)a.n_chunk * rows * g.hd;
  }
  const unsigned ctas = (unsigned)(a.groups * a.n_chunk * g.kv_heads * g.batch);
  magma_status_t st;
  if (dtype == MAGMA_DTYPE_F32) {
    const bool few = a.rows <= 4;
    st = g.hd <= 64 ? (few ? launch_f32<64, 4>(q, k, v, a, ctas, s) : launch_f32<64, 8>(q, k, v, a, ctas, s))
                    : (few ? launch_f32<128, 4>(q, k, v, a, ctas, s) : launch_f32<128, 8>(q, k, v, a, ctas, s));
  } else {
    auto* run = g.hd <= 64 ? (a.rows <= 16 ? launch_bf16<64, 1> : a.rows <= 32 ? launch_bf16<64, 2> : launch_bf16<64, 4>)
                           : (a.rows <= 16 ? launch_bf16<128, 1> : a.rows <= 32 ? launch_bf16<128, 2> : launch_bf16<128, 4>);
    st = run(q, k, v, a, ctas, s);
  }
  if (st || a.part == nullptr) return st;
  return cross_join_parts(a.part, a.part_lse, o, lse, g, a.n_chunk, dtype, s);
}

}  // namespace magma
