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
// The query rows of the heads that share a key head form one list (row =
// shared head * q_len + query), cut into 64-row tiles, so that short queries
// fill a tile together. Everything is bound by the FMA pipe and what feeds it:
// a thread holds a block of products and adds two terms per instruction
// (fma.f32x2): pairs along d for the scores, whose tiles lie in rows of d, and
// pairs along the row index for the second products, whose left operand is
// written to shared memory with that index contiguous. Rows are padded by 16
// bytes, which spreads 16-byte reads of neighbouring rows over the banks. (F32, 8 x 12
// heads of 64, 200 queries over 114 to 333 keys: 57 us, 19.4 of the FMA pipe's 74
// TFLOP/s: 672 CTAs of 32 rows last two to six tiles each, and a tile's loads, maximum
// and exponentials take as long as its products. 2 x 16 heads of 128, 1024 x 1024:
// 508 us, 33.8 TFLOP/s.)
#include <algorithm>
#include <cmath>

#include "cross_attention.cuh"
#include "sm100.cuh"

namespace magma {
namespace {

using u64 = unsigned long long;

constexpr int kRows = 64;       // query rows, and keys of a gradient tile
constexpr int kP = kRows + 4;   // pitch of a tile of probabilities

// A tile of rows: pitch in floats.
template <int HD> constexpr int kPitch = HD + 4;

__device__ __forceinline__ void cp_async16(float* dst, const float* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(sm100::smem_u32(dst)), "l"(src),
               "r"(on ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ROWS rows into dst[ROWS][HD + 4] as F32; `at(r)` is row r's offset from src,
// negative for a row that is not there. Those rows, and columns from hd on,
// become zeros. VEC: F32 rows in 16-byte pieces, asynchronously.
template <int HD, int ROWS, bool VEC, typename T, typename At>
__device__ __forceinline__ void load_rows(float* dst, const T* src, int hd, At at) {
  if constexpr (VEC) {
    constexpr int kPieces = HD / 4;
#pragma unroll 4
    for (int i = threadIdx.x; i < ROWS * kPieces; i += blockDim.x) {
      const int r = i / kPieces, c = i % kPieces * 4;
      const int64_t o = at(r);
      const bool on = o >= 0 && c < hd;
      cp_async16(dst + r * kPitch<HD> + c, src + (on ? o + c : 0), on);
    }
  } else {
    for (int i = threadIdx.x; i < ROWS * HD; i += blockDim.x) {
      const int r = i / HD, c = i % HD;
      const int64_t o = at(r);
      dst[r * kPitch<HD> + c] = o >= 0 && c < hd ? to_f32(src[o + c]) : 0.f;
    }
  }
}

// s[i][j] = sum_d a[row_a(i)][d] b[row_b(j)][d], even and odd d apart.
template <int HD, int NI, int NJ, typename RA, typename RB>
__device__ __forceinline__ void dots(float (&s)[NI][NJ], const float* a, const float* b, RA row_a,
                                     RB row_b) {
  u64 acc[NI][NJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = 0ull;
#pragma unroll 4
  for (int d = 0; d < HD; d += 4) {
    ulonglong2 x[NI], y[NJ];
#pragma unroll
    for (int i = 0; i < NI; ++i)
      x[i] = *reinterpret_cast<const ulonglong2*>(a + row_a(i) * kPitch<HD> + d);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      y[j] = *reinterpret_cast<const ulonglong2*>(b + row_b(j) * kPitch<HD> + d);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        acc[i][j] = f2_fma(x[i].x, y[j].x, acc[i][j]);
        acc[i][j] = f2_fma(x[i].y, y[j].y, acc[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      float lo, hi;
      f2_unpack(acc[i][j], lo, hi);
      s[i][j] = lo + hi;
    }
}

// Column c of a thread's ND columns: groups of four, 64 apart.
__device__ __forceinline__ int col_of(int tx, int c) { return tx * 4 + (c & 3) + 64 * (c >> 2); }

// acc[p][c] += (left pair p) * right[c]: the columns' values doubled into pairs.
template <int NP, int ND>
__device__ __forceinline__ void add_products(u64 (&acc)[NP][ND], const u64 (&left)[NP],
                                             const float* right, int tx) {
#pragma unroll
  for (int q = 0; q < ND / 4; ++q) {
    const float4 v = *reinterpret_cast<const float4*>(right + tx * 4 + 64 * q);
    const u64 w[4] = {f2_pack(v.x, v.x), f2_pack(v.y, v.y), f2_pack(v.z, v.z), f2_pack(v.w, v.w)};
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[p][4 * q + c] = f2_fma(left[p], w[c], acc[p][4 * q + c]);
  }
}

// A CTA's place: tile, key head, sequence, part of the source.
struct Block {
  int64_t tile, kvh, b;
  int part;
};
__device__ __forceinline__ Block block_of(int64_t tiles, int64_t heads, int parts) {
  Block x;
  int64_t i = blockIdx.x;
  x.part = (int)(i % parts);
  i /= parts;
  x.tile = i % tiles;
  x.kvh = i / tiles % heads;
  x.b = i / tiles / heads;
  return x;
}

// The sequence in place i of the sequences by length, the longest first: the CTAs of
// the longest ones, which come last to an end, start first (8 x 12 heads, 200 queries
// over 114 to 333 keys, the shortest first 68 us, the longest first 57; the gradient
// of 4 x 8 heads, 700 over up to 900 keys, as they come 592 and 499 us). Every warp
// finds it by itself; beyond 32 sequences the CTAs are so many that they even out.
__device__ __forceinline__ int64_t longest_first(const CrossGeom& g, int64_t i) {
  if (g.lens == nullptr || g.batch > 32) return i;
  const int lane = threadIdx.x & 31, n = (int)g.batch;
  const int mine = lane < n ? g.lens[lane] : -1;
  int rank = 0;
  for (int o = 0; o < n; ++o) {
    const int other = __shfl_sync(0xffffffffu, mine, o);
    rank += other > mine || (other == mine && o < lane);
  }
  return __ffs(__ballot_sync(0xffffffffu, lane < n && rank == (int)i)) - 1;
}

// Offset of listed query row r of a [B, H, Sq, D] tensor, -1 behind the last.
__device__ __forceinline__ int64_t row_offset(const CrossGeom& g, const Block& x,
                                              const int64_t (&st)[3], int64_t r) {
  if (r >= g.group * g.q_len) return -1;
  return x.b * st[0] + (x.kvh * g.group + r / g.q_len) * st[1] + r % g.q_len * st[2];
}
// Its index in [B, H, Sq].
__device__ __forceinline__ int64_t row_index(const CrossGeom& g, const Block& x, int64_t r) {
  return (x.b * g.heads + x.kvh * g.group + r / g.q_len) * g.q_len + r % g.q_len;
}

// Tiles [t0, t1) of a part.
__device__ __forceinline__ void part_tiles(int64_t tiles, int part, int parts, int64_t& t0,
                                           int64_t& t1) {
  const int64_t each = (tiles + parts - 1) / parts;
  t0 = part * each < tiles ? part * each : tiles;
  t1 = tiles - t0 < each ? tiles : t0 + each;
}

struct FwdArgs {
  CrossGeom g;
  int parts;
  float* part;      // [part][b][h][q][hd] of a split source
  float* part_lse;  // [part][b][h][q]
};

// ------------------------------------------------------------------ forward
// 128 threads; thread (ty, tx) has rows ty 4 + {0..3} and, of a 64-row tile, + 32,
// keys tx + 16 j, columns tx 4 + {0..3} and + 64. K and V of a tile have a buffer
// each: V comes in under the scores, the next K under the sums. 64-row tiles read
// shared memory least (half its bandwidth at the FMA pipe's rate, 32-row tiles
// three quarters); 32-row tiles are for calls that would otherwise not give the
// SMs enough CTAs to even out. Four CTAs per SM (128 registers) where that is
// possible: 2 x 16 heads of 128, 1024 x 1024, 552 -> 509 us; the 32-row tiles of head
// size 64 do better with the 134 registers that they ask for (8 x 12 heads, 200 x
// 114..333: 56.6 and 58.4 us).
template <int HD, int BM>
struct FwdTile {
  static constexpr int kKeys = HD == 64 ? 64 : 32;
  static constexpr int kPp = BM + 4;  // pitch of the probabilities
  static constexpr int kSmem =
      ((BM + 2 * kKeys) * kPitch<HD> + kKeys * kPp) * 4 + BM * 8;
};

template <int HD, int BM, typename T, bool VEC>
__global__ void __launch_bounds__(128, HD == 64 && BM == 32 ? 1 : 4)
cross_fwd(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
          T* __restrict__ o, float* __restrict__ lse, const __grid_constant__ FwdArgs a) {
  constexpr int BN = FwdTile<HD, BM>::kKeys, kP = FwdTile<HD, BM>::kPp;
  constexpr int NI = BM / 8, NP = NI / 2, NK = BN / 16, ND = HD / 16;
  extern __shared__ __align__(16) float sm[];
  float* Qs = sm;
  float* Ks = Qs + BM * kPitch<HD>;
  float* Vs = Ks + BN * kPitch<HD>;
  float* Ps = Vs + BN * kPitch<HD>;                        // [key][row]
  int64_t* offs = reinterpret_cast<int64_t*>(Ps + BN * kP);  // of the query rows
  const CrossGeom& g = a.g;
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const int64_t rows = (int64_t)g.group * g.q_len;
  Block x = block_of((rows + BM - 1) / BM, g.kv_heads, a.parts);
  x.b = longest_first(g, x.b);
  const int64_t r0 = x.tile * BM, len = cross_len(g, x.b);
  int64_t t0, t1;
  part_tiles((len + BN - 1) / BN, x.part, a.parts, t0, t1);
  const T* kh = k + x.b * g.ks[0] + x.kvh * g.ks[1];
  const T* vh = v + x.b * g.vs[0] + x.kvh * g.vs[1];
  auto row = [&](int i) { return ty * 4 + (i & 3) + 32 * (i >> 2); };
  auto load_k = [&](int64_t t) {
    load_rows<HD, BN, VEC>(Ks, kh, g.hd, [&](int r) {
      return t * BN + r < len ? (t * BN + r) * g.ks[2] : (int64_t)-1;
    });
  };
  auto load_v = [&](int64_t t) {
    load_rows<HD, BN, VEC>(Vs, vh, g.hd, [&](int r) {
      return t * BN + r < len ? (t * BN + r) * g.vs[2] : (int64_t)-1;
    });
  };
  if (tid < BM) offs[tid] = row_offset(g, x, g.qs, r0 + tid);
  __syncthreads();
  load_rows<HD, BM, VEC>(Qs, q, g.hd, [&](int r) { return offs[r]; });
  if (t0 < t1) load_k(t0);
  cp_commit();
  u64 acc[NP][ND];
  float m[NI], l[NI];
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int c = 0; c < ND; ++c) acc[p][c] = 0ull;
#pragma unroll
  for (int i = 0; i < NI; ++i) m[i] = -INFINITY, l[i] = 0.f;
  for (int64_t t = t0; t < t1; ++t) {
    cp_wait<0>();
    __syncthreads();  // K is there; the last tile's V and P have been used
    load_v(t);
    cp_commit();
    float s[NI][NK];
    dots<HD>(s, Qs, Ks, row, [&](int j) { return tx + 16 * j; });
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NK; ++j) s[i][j] *= g.scale;
    if (len - t * BN < BN) {  // the thread's keys that are not there
      const int left = (int)(len - t * BN) - tx;
#pragma unroll
      for (int j = 0; j < NK; ++j)
#pragma unroll
        for (int i = 0; i < NI; ++i)
          if (16 * j >= left) s[i][j] = -INFINITY;
    }
    float alpha[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < NK; ++j) mx = fmaxf(mx, s[i][j]);
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
      const float mn = fmaxf(m[i], mx);
      const float ref = mn == -INFINITY ? 0.f : mn;  // a row of -inf scores
      alpha[i] = expf(m[i] - ref);
      m[i] = mn;
      float rs = 0.f;
#pragma unroll
      for (int j = 0; j < NK; ++j) {
        s[i][j] = expf(s[i][j] - ref);
        rs += s[i][j];
      }
      l[i] = l[i] * alpha[i] + rs;  // the thread's keys; the 16 threads meet at the end
    }
#pragma unroll
    for (int j = 0; j < NK; ++j)
#pragma unroll
      for (int h = 0; h < NI / 4; ++h)
        *reinterpret_cast<float4*>(Ps + (tx + 16 * j) * kP + ty * 4 + 32 * h) =
            make_float4(s[4 * h][j], s[4 * h + 1][j], s[4 * h + 2][j], s[4 * h + 3][j]);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const u64 f = f2_pack(alpha[2 * p], alpha[2 * p + 1]);
#pragma unroll
      for (int c = 0; c < ND; ++c) acc[p][c] = f2_mul(acc[p][c], f);
    }
    cp_wait<0>();
    __syncthreads();  // V and P are there; K has been used
    if (t + 1 < t1) load_k(t + 1);
    cp_commit();
#pragma unroll 4
    for (int key = 0; key < BN; ++key) {
      u64 left[NP];
#pragma unroll
      for (int h = 0; h < NI / 4; ++h) {
        const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(Ps + key * kP + ty * 4 + 32 * h);
        left[2 * h] = x.x;
        left[2 * h + 1] = x.y;
      }
      add_products(acc, left, Vs + key * kPitch<HD>, tx);
    }
  }
  cp_wait<0>();
  const int64_t all = g.batch * g.heads * g.q_len;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
    const int64_t r = r0 + row(i);
    if (r >= rows) continue;
    const float inv = l[i] == 0.f ? 0.f : 1.0f / l[i];  // no keys: a zero row
    const float out_lse = l[i] == 0.f ? -INFINITY : m[i] + logf(l[i]);
    const int64_t at = row_index(g, x, r);
    if (a.parts > 1) {
      if (tx == 0) a.part_lse[x.part * all + at] = out_lse;
    } else if (tx == 0 && lse != nullptr) {
      lse[at] = out_lse;
    }
    const int64_t oo = row_offset(g, x, g.os, r);
#pragma unroll
    for (int c = 0; c < ND; ++c) {
      float lo, hi;
      f2_unpack(acc[i >> 1][c], lo, hi);
      const float y = (i & 1 ? hi : lo) * inv;
      const int d = col_of(tx, c);
      if (d >= g.hd) continue;
      if (a.parts > 1) a.part[(x.part * all + at) * g.hd + d] = y;
      else o[oo + d] = from_f32<T>(y);
    }
  }
}

// delta[b, h, i] = sum_d dO[i, d] * O[i, d]; one warp per row.
template <typename T>
__global__ void __launch_bounds__(256)
cross_delta(const T* __restrict__ o, const T* __restrict__ d_o, float* __restrict__ delta,
            const CrossGeom g) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = g.batch * g.heads * g.q_len;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows;
       r += (int64_t)gridDim.x * 8) {
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

// The terms of the query rows of a tile: lse and delta, (inf, 0) behind the last.
__device__ __forceinline__ void row_terms(const CrossGeom& g, const Block& x, int64_t r,
                                          const float* lse, const float* delta, float& l, float& e) {
  const bool on = r < (int64_t)g.group * g.q_len;
  const int64_t at = on ? row_index(g, x, r) : 0;
  l = on ? row_lse(lse[at]) : INFINITY;
  e = on ? delta[at] : 0.f;
}

// P and dS of a row's four keys from the dot products; a key from len on takes no
// part, a query row that is not there has lse = inf. Where the tile has all keys
// of the row (`whole`; the 16 threads of a row are half a warp), delta is formed
// from P and dP: the stored O is rounded to the tensor's type, and a few keys do
// not average that out.
template <typename On>
__device__ __forceinline__ void probs(float (&s)[4], float (&dp)[4], On on, float scale, float lse,
                                      float delta, bool whole) {
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    s[j] = on(j) ? expf(s[j] * scale - lse) : 0.f;
    if (on(j)) sum = fmaf(s[j], dp[j], sum);
  }
  if (whole) {
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    delta = sum;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) dp[j] = on(j) ? s[j] * (dp[j] - delta) : 0.f;
}

// Where few tiles have many steps, a tile's steps are split into parts, whose F32
// sums are added up in order by cross_sum.
struct BwdArgs {
  CrossGeom g;
  int kv_parts, q_parts;  // of the query rows in dK and dV, of the keys in dQ
  float* part;            // [part][dV, dK][b][kvh][key][hd], or [part][b][h][q][hd]
};

// --------------------------------------------------------------- dK and dV
// One CTA of 256 threads per (key tile, key head, sequence). Scores: thread (ty,
// tx) has rows ty 4 + {0..3}, keys tx + 16 j. Sums: keys ty 4 + {0..3}, columns
// as above.
template <int HD> constexpr int kDkvSmem = (4 * kRows * kPitch<HD> + 2 * kRows * kP + 2 * kRows) * 4 + 2 * kRows * 8;

template <int HD, typename T, bool VEC>
__global__ void __launch_bounds__(256, HD == 64 ? 2 : 1)
cross_dkdv(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
           const T* __restrict__ d_o, const float* __restrict__ lse,
           const float* __restrict__ delta, T* __restrict__ dk, T* __restrict__ dv,
           const __grid_constant__ BwdArgs a) {
  const CrossGeom& g = a.g;
  constexpr int ND = HD / 16;
  extern __shared__ __align__(16) float sm[];
  float* Ks = sm;
  float* Vs = Ks + kRows * kPitch<HD>;
  float* Qs = Vs + kRows * kPitch<HD>;
  float* Gs = Qs + kRows * kPitch<HD>;  // dO
  float* Ps = Gs + kRows * kPitch<HD>;  // [row][key]
  float* Ds = Ps + kRows * kP;          // dS, [row][key]
  float* Ls = Ds + kRows * kP;          // lse of the query rows
  float* Es = Ls + kRows;               // delta
  int64_t* qo = reinterpret_cast<int64_t*>(Es + kRows);
  int64_t* go = qo + kRows;
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const Block x = block_of((g.kv_len + kRows - 1) / kRows, g.kv_heads, a.kv_parts);
  const int64_t k0 = x.tile * kRows, len = cross_len(g, x.b);
  const int64_t rows = (int64_t)g.group * g.q_len;
  int64_t t0, t1;
  part_tiles((rows + kRows - 1) / kRows, x.part, a.kv_parts, t0, t1);
  u64 adk[2][ND], adv[2][ND];
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int c = 0; c < ND; ++c) adk[p][c] = adv[p][c] = 0ull;
  if (k0 < len) {
    auto key = [&](int64_t st) {
      return [&g, k0, len, st](int r) { return k0 + r < len ? (k0 + r) * st : (int64_t)-1; };
    };
    load_rows<HD, kRows, VEC>(Ks, k + x.b * g.ks[0] + x.kvh * g.ks[1], g.hd, key(g.ks[2]));
    load_rows<HD, kRows, VEC>(Vs, v + x.b * g.vs[0] + x.kvh * g.vs[1], g.hd, key(g.vs[2]));
    for (int64_t r0 = t0 * kRows; r0 < t1 * kRows; r0 += kRows) {
      __syncthreads();
      if (tid < kRows) {
        qo[tid] = row_offset(g, x, g.qs, r0 + tid);
        go[tid] = row_offset(g, x, g.dos, r0 + tid);
        row_terms(g, x, r0 + tid, lse, delta, Ls[tid], Es[tid]);
      }
      __syncthreads();
      load_rows<HD, kRows, VEC>(Qs, q, g.hd, [&](int r) { return qo[r]; });
      load_rows<HD, kRows, VEC>(Gs, d_o, g.hd, [&](int r) { return go[r]; });
      cp_commit();
      cp_wait<0>();
      __syncthreads();
      float s[4][4], dp[4][4];
      auto row = [&](int i) { return ty * 4 + i; };
      auto col = [&](int j) { return tx + 16 * j; };
      dots<HD>(s, Qs, Ks, row, col);
      dots<HD>(dp, Gs, Vs, row, col);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = row(i);
        probs(s[i], dp[i], [&](int j) { return k0 + col(j) < len; }, g.scale, Ls[r], Es[r],
              len <= kRows);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          Ps[r * kP + col(j)] = s[i][j];
          Ds[r * kP + col(j)] = dp[i][j];
        }
      }
      __syncthreads();
#pragma unroll 4
      for (int r = 0; r < kRows; ++r) {
        const ulonglong2 p = *reinterpret_cast<const ulonglong2*>(Ps + r * kP + ty * 4);
        const ulonglong2 d = *reinterpret_cast<const ulonglong2*>(Ds + r * kP + ty * 4);
        const u64 lp[2] = {p.x, p.y}, ld[2] = {d.x, d.y};
        add_products(adv, lp, Gs + r * kPitch<HD>, tx);
        add_products(adk, ld, Qs + r * kPitch<HD>, tx);
      }
    }
  }
  cp_wait<0>();
  T* dkh = dk + x.b * g.dks[0] + x.kvh * g.dks[1];
  T* dvh = dv + x.b * g.dvs[0] + x.kvh * g.dvs[1];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t kj = k0 + ty * 4 + i;
    if (kj >= g.kv_len) continue;
#pragma unroll
    for (int c = 0; c < ND; ++c) {
      const int d = col_of(tx, c);
      if (d >= g.hd) continue;
      float a0, a1, b0, b1;
      f2_unpack(adk[i >> 1][c], a0, a1);
      f2_unpack(adv[i >> 1][c], b0, b1);
      if (a.kv_parts > 1) {
        const int64_t all = g.batch * g.kv_heads * g.kv_len * g.hd;
        const int64_t at = ((x.b * g.kv_heads + x.kvh) * g.kv_len + kj) * g.hd + d;
        a.part[2 * x.part * all + at] = i & 1 ? b1 : b0;
        a.part[(2 * x.part + 1) * all + at] = i & 1 ? a1 : a0;
        continue;
      }
      dkh[kj * g.dks[2] + d] = from_f32<T>((i & 1 ? a1 : a0) * g.scale);
      dvh[kj * g.dvs[2] + d] = from_f32<T>(i & 1 ? b1 : b0);
    }
  }
}

// ---------------------------------------------------------------------- dQ
// One CTA of 256 threads per (row tile, key head, sequence); sums: rows ty 4 +
// {0..3}, columns as above.
template <int HD> constexpr int kDqSmem = (4 * kRows * kPitch<HD> + kRows * kP) * 4 + 2 * kRows * 8;

template <int HD, typename T, bool VEC>
__global__ void __launch_bounds__(256, HD == 64 ? 2 : 1)
cross_dq(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
         const T* __restrict__ d_o, const float* __restrict__ lse,
         const float* __restrict__ delta, T* __restrict__ dq, const __grid_constant__ BwdArgs a) {
  const CrossGeom& g = a.g;
  constexpr int ND = HD / 16;
  extern __shared__ __align__(16) float sm[];
  float* Qs = sm;
  float* Gs = Qs + kRows * kPitch<HD>;
  float* Ks = Gs + kRows * kPitch<HD>;
  float* Vs = Ks + kRows * kPitch<HD>;
  float* Ds = Vs + kRows * kPitch<HD>;  // dS, [key][row]
  int64_t* qo = reinterpret_cast<int64_t*>(Ds + kRows * kP);
  int64_t* go = qo + kRows;
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const int64_t rows = (int64_t)g.group * g.q_len;
  Block x = block_of((rows + kRows - 1) / kRows, g.kv_heads, a.q_parts);
  x.b = longest_first(g, x.b);
  const int64_t r0 = x.tile * kRows, len = cross_len(g, x.b);
  int64_t t0, t1;
  part_tiles((len + kRows - 1) / kRows, x.part, a.q_parts, t0, t1);
  const T* kh = k + x.b * g.ks[0] + x.kvh * g.ks[1];
  const T* vh = v + x.b * g.vs[0] + x.kvh * g.vs[1];
  if (tid < kRows) {
    qo[tid] = row_offset(g, x, g.qs, r0 + tid);
    go[tid] = row_offset(g, x, g.dos, r0 + tid);
  }
  __syncthreads();
  load_rows<HD, kRows, VEC>(Qs, q, g.hd, [&](int r) { return qo[r]; });
  load_rows<HD, kRows, VEC>(Gs, d_o, g.hd, [&](int r) { return go[r]; });
  auto row = [&](int i) { return ty * 4 + i; };
  auto col = [&](int j) { return tx + 16 * j; };
  float ls[4], es[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) row_terms(g, x, r0 + row(i), lse, delta, ls[i], es[i]);
  u64 acc[2][ND];
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int c = 0; c < ND; ++c) acc[p][c] = 0ull;
  for (int64_t k0 = t0 * kRows; k0 < t1 * kRows; k0 += kRows) {
    __syncthreads();
    auto key = [&](int64_t st) {
      return [&g, k0, len, st](int r) { return k0 + r < len ? (k0 + r) * st : (int64_t)-1; };
    };
    load_rows<HD, kRows, VEC>(Ks, kh, g.hd, key(g.ks[2]));
    load_rows<HD, kRows, VEC>(Vs, vh, g.hd, key(g.vs[2]));
    cp_commit();
    cp_wait<0>();
    __syncthreads();
    float s[4][4], dp[4][4];
    dots<HD>(s, Qs, Ks, row, col);
    dots<HD>(dp, Gs, Vs, row, col);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      probs(s[i], dp[i], [&](int j) { return k0 + col(j) < len; }, g.scale, ls[i], es[i],
            len <= kRows);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      *reinterpret_cast<float4*>(Ds + col(j) * kP + ty * 4) =
          make_float4(dp[0][j], dp[1][j], dp[2][j], dp[3][j]);
    }
    __syncthreads();
#pragma unroll 4
    for (int c = 0; c < kRows; ++c) {
      const ulonglong2 d = *reinterpret_cast<const ulonglong2*>(Ds + c * kP + ty * 4);
      const u64 left[2] = {d.x, d.y};
      add_products(acc, left, Ks + c * kPitch<HD>, tx);
    }
  }
  cp_wait<0>();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t o = row_offset(g, x, g.dqs, r0 + row(i));
    if (o < 0) continue;
#pragma unroll
    for (int c = 0; c < ND; ++c) {
      const int d = col_of(tx, c);
      if (d >= g.hd) continue;
      float lo, hi;
      f2_unpack(acc[i >> 1][c], lo, hi);
      const float y = i & 1 ? hi : lo;
      if (a.q_parts > 1)
        a.part[(x.part * g.batch * g.heads * g.q_len + row_index(g, x, r0 + row(i))) * g.hd + d] = y;
      else
        dq[o + d] = from_f32<T>(y * g.scale);
    }
  }
}

// out[b][h][n][d] = mul * sum over the parts, in order; `step`: elements from a part
// to the next.
struct SumArgs {
  const float* part;
  int64_t step, heads, n, total;
  int64_t st[3];
  int parts, hd;
  float mul;
};
template <typename T>
__global__ void __launch_bounds__(256) cross_sum(const SumArgs a, T* __restrict__ out) {
  wait_for_launch_before();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.total;
       i += (int64_t)gridDim.x * 256) {
    float s = 0.f;
#pragma unroll 4
    for (int p = 0; p < a.parts; ++p) s += a.part[p * a.step + i];
    const int64_t row = i / a.hd, n = row % a.n, bh = row / a.n;
    out[bh / a.heads * a.st[0] + bh % a.heads * a.st[1] + n * a.st[2] + i % a.hd] =
        from_f32<T>(s * a.mul);
  }
}

// ---------------------------------------------------------------- host side
magma_status_t blocks_of(int64_t tiles, int64_t heads, int64_t batch, int64_t parts, unsigned* n) {
  const double all = (double)tiles * (double)heads * (double)batch * (double)parts;
  if (all > 2147483647.0)
    return fail(MAGMA_INVALID_ARGUMENT, "cross attention: more than 2^31 - 1 tiles");
  *n = (unsigned)(tiles * heads * batch * parts);
  return MAGMA_OK;
}

int64_t row_tiles(const CrossGeom& g, int rows = kRows) {
  return ceil_div((int64_t)g.group * g.q_len, rows);
}

// Rows in 16-byte pieces.
bool pieces(const void* p, const int64_t (&st)[3]) {
  return aligned16(p) && st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] % 4 == 0;
}

// Rows of a forward tile: 32 where 64-row tiles would be fewer than four per SM
// (8 x 12 heads of 64, 200 queries over 114 to 333 keys: 57 us; before the
// longest came first 59 to 63, and with 64 rows 68 to 73).
int fwd_rows(const CrossGeom& g) {
  return row_tiles(g) * g.kv_heads * g.batch < 4LL * num_sms() ? 32 : 64;
}

template <int HD, int BM, typename T, bool VEC>
magma_status_t fwd_rows_of(const void* q, const void* k, const void* v, void* o, float* lse,
                           const FwdArgs& a, cudaStream_t s) {
  const CrossGeom& g = a.g;
  constexpr int smem = FwdTile<HD, BM>::kSmem;
  unsigned n;
  if (magma_status_t st = cross_smem<cross_fwd<HD, BM, T, VEC>>(smem)) return st;
  if (magma_status_t st = blocks_of(row_tiles(g, BM), g.kv_heads, g.batch, a.parts, &n)) return st;
  cross_fwd<HD, BM, T, VEC><<<n, 128, smem, s>>>((const T*)q, (const T*)k, (const T*)v, (T*)o, lse, a);
  return check_launch("cross_fwd");
}
template <int HD, typename T, bool VEC>
magma_status_t fwd(const void* q, const void* k, const void* v, void* o, float* lse,
                   const FwdArgs& a, cudaStream_t s) {
  return fwd_rows(a.g) == 32 ? fwd_rows_of<HD, 32, T, VEC>(q, k, v, o, lse, a, s)
                             : fwd_rows_of<HD, 64, T, VEC>(q, k, v, o, lse, a, s);
}

// Parts of a tile's steps where the tiles do not give every SM two CTAs: as many as
// give it four, of at least two steps. (Gradients in F32, whole, in parts for two CTAs
// per SM, and for four: 8 heads over 2 of 64, 40 x 3000, 407, 70 and 70 us; 8 heads, 200 x
// 333, 97, 55 and 55; 6 x 8 heads, 256 x 512, 226, 226 and 213; 4 heads of 128, 1024 x
// 1024, 478, 286 and 320. With CTAs for most SMs already the parts cost more than they
// give: 4 x 8 heads of 64, 512 x 512, 252, 252 and 288.)
int64_t grad_parts(int64_t ctas, int64_t steps) {
  if (ctas >= 2 * num_sms()) return 1;
  return std::max<int64_t>(1, std::min<int64_t>(4LL * num_sms() / std::max<int64_t>(ctas, 1), steps / 2));
}
int64_t kv_parts(const CrossGeom& g) {
  return grad_parts(ceil_div(g.kv_len, kRows) * g.kv_heads * g.batch, row_tiles(g));
}
int64_t q_parts(const CrossGeom& g) {
  return grad_parts(row_tiles(g) * g.kv_heads * g.batch, ceil_div(g.kv_len, kRows));
}
size_t kv_part_bytes(const CrossGeom& g) {
  return 2 * sizeof(float) * (size_t)g.batch * g.kv_heads * g.kv_len * g.hd;
}
size_t q_part_bytes(const CrossGeom& g) {
  return sizeof(float) * (size_t)g.batch * g.heads * g.q_len * g.hd;
}
size_t delta_bytes(const CrossGeom& g) {
  return (sizeof(float) * (size_t)g.batch * g.heads * g.q_len + 15) / 16 * 16;
}

template <typename T>
magma_status_t sum_parts(const float* part, int64_t step, int64_t parts, int64_t batch, int64_t heads,
                         int64_t n, int hd, const int64_t (&st)[3], float mul, void* out,
                         cudaStream_t s) {
  SumArgs a{part, step, heads, n, batch * heads * n * hd, {st[0], st[1], st[2]}, (int)parts, hd, mul};
  const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(a.total, 256), 8LL * num_sms());
  return launch_after(cross_sum<T>, dim3(blocks), 256, 0, s, "cross_sum", a, static_cast<T*>(out));
}

template <int HD, typename T, bool VEC>
magma_status_t bwd(const void* q, const void* k, const void* v, const void* o, const void* d_o,
                   const float* lse, void* dq, void* dk, void* dv, float* delta, const BwdArgs& a,
                   cudaStream_t s) {
  const CrossGeom& g = a.g;
  if (magma_status_t st = cross_smem<cross_dkdv<HD, T, VEC>>(kDkvSmem<HD>)) return st;
  if (magma_status_t st = cross_smem<cross_dq<HD, T, VEC>>(kDqSmem<HD>)) return st;
  unsigned nq = 0, nk = 0;
  if (magma_status_t st = blocks_of(row_tiles(g), g.kv_heads, g.batch, a.q_parts, &nq)) return st;
  if (magma_status_t st = blocks_of(ceil_div(g.kv_len, kRows), g.kv_heads, g.batch, a.kv_parts, &nk)) return st;
  if (nq > 0) {
    const int64_t cap = 16LL * num_sms();
    const int64_t nd = ceil_div(g.batch * g.heads * g.q_len, 8);
    cross_delta<T><<<(unsigned)std::min(cap, nd), 256, 0, s>>>((const T*)o, (const T*)d_o, delta, g);
    if (magma_status_t st = check_launch("cross_delta")) return st;
  }
  if (nk > 0) {
    cross_dkdv<HD, T, VEC><<<nk, 256, kDkvSmem<HD>, s>>>((const T*)q, (const T*)k, (const T*)v,
                                                         (const T*)d_o, lse, delta, (T*)dk, (T*)dv, a);
    if (magma_status_t st = check_launch("cross_dkdv")) return st;
    if (a.kv_parts > 1) {
      const int64_t all = g.batch * g.kv_heads * g.kv_len * g.hd;
      if (magma_status_t st = sum_parts<T>(a.part, 2 * all, a.kv_parts, g.batch, g.kv_heads, g.kv_len,
                                           g.hd, g.dvs, 1.f, dv, s))
        return st;
      if (magma_status_t st = sum_parts<T>(a.part + all, 2 * all, a.kv_parts, g.batch, g.kv_heads,
                                           g.kv_len, g.hd, g.dks, g.scale, dk, s))
        return st;
    }
  }
  if (nq > 0) {
    cross_dq<HD, T, VEC><<<nq, 256, kDqSmem<HD>, s>>>((const T*)q, (const T*)k, (const T*)v,
                                                      (const T*)d_o, lse, delta, (T*)dq, a);
    if (magma_status_t st = check_launch("cross_dq")) return st;
    if (a.q_parts > 1)
      return sum_parts<T>(a.part, g.batch * g.heads * g.q_len * g.hd, a.q_parts, g.batch, g.heads,
                          g.q_len, g.hd, g.dqs, g.scale, dq, s);
  }
  return MAGMA_OK;
}

// Parts of a source where the tiles do not give every SM four CTAs: as many as
// give it six, of at least two tiles. (8 x 12 heads, 200 queries, 333 keys: 384
// tiles take 73 us whole and 84 us in two parts each; 8 heads over 2, 40 queries,
// 3000 keys: 42 us in 11 parts of four tiles, 34 us in 23 of two.)
int64_t wanted_parts(const CrossGeom& g) {
  const int64_t ctas = std::max<int64_t>(row_tiles(g, fwd_rows(g)) * g.kv_heads * g.batch, 1);
  const int64_t tiles = ceil_div(g.kv_len, g.hd <= 64 ? 64 : 32);
  if (ctas >= 4 * num_sms()) return 1;
  return std::max<int64_t>(1, std::min<int64_t>(6LL * num_sms() / ctas, tiles / 2));
}

}  // namespace

size_t cross_simt_fwd_workspace(const CrossGeom& g) {
  const int64_t n = g.hd % 4 == 0 ? wanted_parts(g) : 1;
  return n <= 1 ? 0 : (size_t)n * g.batch * g.heads * g.q_len * (g.hd + 1) * sizeof(float);
}

magma_status_t cross_fwd_simt(const void* q, const void* k, const void* v, void* o, float* lse,
                              const CrossGeom& g, magma_dtype_t dtype, void* workspace,
                              size_t workspace_bytes, cudaStream_t s) {
  FwdArgs a{};
  a.g = g;
  a.parts = 1;
  const int64_t rows = g.batch * g.heads * g.q_len;
  const size_t each = (size_t)rows * (g.hd + 1) * sizeof(float);
  const bool join_ok = g.hd % 4 == 0 && g.os[0] % 4 == 0 && g.os[1] % 4 == 0 && g.os[2] % 4 == 0 &&
                       aligned16(o);
  if (workspace != nullptr && aligned16(workspace) && join_ok)
    a.parts = (int)std::max<int64_t>(1, std::min<int64_t>(wanted_parts(g), workspace_bytes / each));
  if (a.parts > 1) {
    a.part = static_cast<float*>(workspace);
    a.part_lse = a.part + (size_t)a.parts * rows * g.hd;
  }
  const bool vec = dtype == MAGMA_DTYPE_F32 && g.hd % 4 == 0 && pieces(q, g.qs) &&
                   pieces(k, g.ks) && pieces(v, g.vs);
  magma_status_t st;
  if (dtype == MAGMA_DTYPE_F32)
    st = g.hd <= 64 ? (vec ? fwd<64, float, true>(q, k, v, o, lse, a, s) : fwd<64, float, false>(q, k, v, o, lse, a, s))
                    : (vec ? fwd<128, float, true>(q, k, v, o, lse, a, s) : fwd<128, float, false>(q, k, v, o, lse, a, s));
  else
    st = g.hd <= 64 ? fwd<64, __nv_bfloat16, false>(q, k, v, o, lse, a, s)
                    : fwd<128, __nv_bfloat16, false>(q, k, v, o, lse, a, s);
  if (st || a.parts == 1) return st;
  return cross_join_parts(a.part, a.part_lse, o, lse, g, a.parts, dtype, s);
}

size_t cross_simt_bwd_workspace(const CrossGeom& g) {
  const int64_t nk = kv_parts(g), nq = q_parts(g);
  return delta_bytes(g) + std::max(nk > 1 ? nk * kv_part_bytes(g) : 0, nq > 1 ? nq * q_part_bytes(g) : 0);
}

magma_status_t cross_bwd_simt(const void* q, const void* k, const void* v, const void* o,
                              const void* d_o, const float* lse, void* dq, void* dk, void* dv,
                              const CrossGeom& g, magma_dtype_t dtype, void* workspace,
                              size_t workspace_bytes, cudaStream_t s) {
  float* delta = static_cast<float*>(workspace);
  BwdArgs a{};
  a.g = g;
  a.kv_parts = a.q_parts = 1;
  if (workspace_bytes > delta_bytes(g)) {
    const size_t room = workspace_bytes - delta_bytes(g);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + delta_bytes(g));
    if (const size_t each = kv_part_bytes(g))
      a.kv_parts = (int)std::max<int64_t>(1, std::min<int64_t>(kv_parts(g), room / each));
    if (const size_t each = q_part_bytes(g))
      a.q_parts = (int)std::max<int64_t>(1, std::min<int64_t>(q_parts(g), room / each));
  }
  const bool vec = dtype == MAGMA_DTYPE_F32 && g.hd % 4 == 0 && pieces(q, g.qs) &&
                   pieces(k, g.ks) && pieces(v, g.vs) && pieces(d_o, g.dos);
  if (dtype == MAGMA_DTYPE_F32)
    return g.hd <= 64 ? (vec ? bwd<64, float, true>(q, k, v, o, d_o, lse, dq, dk, dv, delta, a, s)
                             : bwd<64, float, false>(q, k, v, o, d_o, lse, dq, dk, dv, delta, a, s))
                      : (vec ? bwd<128, float, true>(q, k, v, o, d_o, lse, dq, dk, dv, delta, a, s)
                             : bwd<128, float, false>(q, k, v, o, d_o, lse, dq, dk, dv, delta, a, s));
  return g.hd <= 64 ? bwd<64, __nv_bfloat16, false>(q, k, v, o, d_o, lse, dq, dk, dv, delta, a, s)
                    : bwd<128, __nv_bfloat16, false>(q, k, v, o, d_o, lse, dq, dk, dv, delta, a, s);
}

}  // namespace magma
