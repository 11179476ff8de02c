// Attention of queries over the keys and values of another sequence on the
// tcgen05 tensor cores: BF16, F32 accumulation, head sizes that are multiples
// of 8 up to 128, padded to 64 or 128 columns by the tensor maps' zero fill. The
// products run over the padded columns, so that their counts are constants: sizes
// between cost almost what the next of the two does (8 x 16 heads, 512 queries, 1024
// keys, forward and gradient: 32 columns 33 and 91 us, 64 35 and 101, 80 39 and 133, 96
// 40 and 136, 128 41 and 142).
//
//   cross_fwd_tc     O_t += P_t V_j over the key tiles j, S_t = Q_t K_j^T
//   cross_rows       -lse log2(e) and delta = rowsum(dO O) of every query row
//   cross_dq_tc      dQ_t += dS_t K_j over the key tiles
//   cross_dkdv_tc    dV += P^T dO, dK += dS^T Q over the query tiles of every
//                    head that shares the key head
//   cross_dq_join, cross_dkdv_join  the pieces of the sums that two CTAs shared
//
// Formulas as in cross_attention_simt.cu. The gradient recomputes S and dP in
// both of its passes (14 instead of 10 products of the size of S) and needs no
// atomics: an output element is added up by one CTA, or in pieces that a join
// adds in a fixed order, so the result is the same on every run.
//
// All three products kernels have the same frame: persistent, one CTA per SM, a
// TMA warp, a warp with one elected lane that issues the MMAs (elect.sync, not
// lane == 0: with it the compiler keeps descriptors and barriers in uniform
// registers; the gradient of 2 x 32 heads of 128, 2048 queries, 4096 keys, 1233 ->
// 924 us), and
// two warpgroups (thread = row) that turn score tiles into probabilities; while
// one works the tensor cores run for the other. Lengths that differ between the sequences are dealt
// out longest first in a snake over the CTAs. Rows of V (forward) or K (dQ) from
// the length on are set to zero in shared memory before a product reads them,
// so whatever lies behind a length meets a probability of 0 only as 0.
//
// What bounds them. Forward of 4 x 32 heads over 8 of size 128, 2048 queries, up to
// 4096 keys: 324 to 331 us, 1.2 PFLOP/s, what the tensor cores' power limit leaves
// (385 us when it is repeated for seconds); head size 64: 275 to 295 us, bound by
// the exponentials, which are as many for half the products. Gradient of 2 x 32
// heads over 8 of size 128, 2048 queries, 4096 keys: 800 to 850 us (rows 16, dQ 350
// and its join 17, dK and dV 430 and 13), 0.83 PFLOP/s of the 10 products that are
// needed, 1.16 of the 14 that are done. 8 x 16 heads of 64, 512 queries, up to 1024
// keys: 80 us (rows 7, dQ 38, dK and dV 48 alone; each begins beside the end of the one
// before it, without that 84). There a 64-query step takes some 1250
// cycles where its products take 700: the issuing lane's waits and the warpgroups'
// chain S -> P -> dS. Two issuing warps (S, P^T and dV; dP, dS^T and dK), three score
// buffers, four warpgroups of 32 columns, warpgroups that take turns at the
// exponentials took 2 to 7 us more.
#include <cuda.h>

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "cross_attention.cuh"
#include "sm100.cuh"

namespace magma {
namespace {

using namespace sm100;

constexpr int kRows = 128;            // query rows of a tile, keys of a forward tile
constexpr int kThreads = 320;         // two warpgroups, TMA warp, MMA warp
constexpr int kTmaWarp = 8, kMmaWarp = 9;
constexpr int kOrder = 512;           // sequences that are dealt out by length
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRescaleLog2 = 8.0f;
constexpr int kBlk128 = 128 * 128;    // bytes of 64 columns of a 128-row tile
constexpr int kBlk64 = 64 * 128;      // and of a 64-row tile

// The exponent's scale in base 2. A scale of 0 becomes the smallest normal
// number: products of finite scores with it leave every exponential at 1, and a
// masked score of -inf still gives 0.
__device__ __forceinline__ float scale_log2(float scale) { return fmaxf(scale * kLog2e, 1.17549435e-38f); }

struct TcArgs {
  CrossGeom g;
  int n_qt;                 // 128-row query tiles of a head
  int n_pairs;              // pairs of (head, query tile) of a key head
  int n_split;
  int q_pad;                // query rows padded to 64 in nlse and delta
  // 0 where a tensor's batch or head stride is 0: its map has one entry there
  int qb, qh, kb, kh, vb, vh, db, dh;
  void* o;
  float* lse;
  float* part;              // [split][b][h][q][hd] of a split source
  float* part_lse;          // [split][b][h][q]
  const float* nlse;        // [b][h][q_pad], -lse log2(e)
  float* delta;             // [b][h][q_pad], rowsum(dO O)
  float* piece;             // partial sums of units that several CTAs share, or NULL
  // dK and dV may begin while dQ is ending: the row terms are there by then
  int early;
  void* dq;
  void* dk;
  void* dv;
};

// True in one lane of a converged warp. The compiler knows that a single lane
// runs what depends on it, and keeps the operands of the MMAs and copies issued
// there in uniform registers (with `lane == 0` it serialises over the lanes).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

// A K-major operand: rows of 128 bytes, eight rows an atom.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) { return smem_desc_sw128(addr, 16, 1024); }
// An MN-major operand whose 64-column blocks are `blk` bytes apart.
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t blk) {
  return smem_desc_sw128(addr, blk, 1024);
}
// The start address is in 16-byte units in the low bits and never carries.
__device__ __forceinline__ uint64_t desc_add(uint64_t d, uint32_t bytes) {
  return d + (uint64_t)(bytes >> 4);
}
// Byte offset of columns [16 kk, 16 kk + 16) of a K-major tile.
__device__ __forceinline__ constexpr uint32_t k_step(int kk, int blk) {
  return (uint32_t)((kk >> 2) * blk + (kk & 3) * 32);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t align1024(uint8_t* raw, uint8_t** p) {
  const uint32_t a = smem_u32(raw);
  const uint32_t base = (a + 1023u) & ~1023u;
  *p = raw + (base - a);
  return base;
}

// The r-th unit of CTA c among n CTAs, even rounds in CTA order, odd ones
// reversed; -1 past the end.
__device__ __forceinline__ int snake(int r, int c, int n, int units) {
  const int64_t u = (int64_t)r * n + ((r & 1) ? n - 1 - c : c);
  return u < units ? (int)u : -1;
}

// order[rank] = sequence, longest first.
__device__ __forceinline__ void order_by_length(const CrossGeom& g, uint16_t* order) {
  if (g.lens == nullptr || g.batch > kOrder) return;
  for (int i = threadIdx.x; i < (int)g.batch; i += blockDim.x) {
    const int n = g.lens[i];
    int rank = 0;
    for (int j = 0; j < (int)g.batch; ++j) {
      const int o = g.lens[j];
      rank += o > n || (o == n && j < i);
    }
    order[rank] = (uint16_t)i;
  }
}
__device__ __forceinline__ int sequence_of(const CrossGeom& g, const uint16_t* order, int rank) {
  return g.lens == nullptr || g.batch > kOrder ? rank : order[rank];
}

// Sets row r of a tile to zero: `blocks` blocks of 128 bytes, `blk` apart.
__device__ __forceinline__ void zero_row(uint32_t tile, int r, int blocks, int blk) {
  for (int i = 0; i < blocks; ++i)
#pragma unroll
    for (int c = 0; c < 8; ++c)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + i * blk + r * 128 + c * 16),
                   "r"(0u)
                   : "memory");
}

// 32 F32 columns of a row times mul as BF16, those below `cols`. A thread has a
// row: 32-byte stores fill whole sectors, where the row's address allows them.
__device__ __forceinline__ void store_cols32(__nv_bfloat16* dst, const uint32_t (&v)[32], float mul,
                                             int cols) {
  uint32_t u[16];
#pragma unroll
  for (int e = 0; e < 16; ++e)
    u[e] = pack_bf16(__uint_as_float(v[2 * e]) * mul, __uint_as_float(v[2 * e + 1]) * mul);
  if ((reinterpret_cast<uintptr_t>(dst) & 31u) == 0 && cols % 16 == 0) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
      if (q * 16 < cols)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + 16 * q),
                     "r"(u[8 * q]), "r"(u[8 * q + 1]), "r"(u[8 * q + 2]), "r"(u[8 * q + 3]),
                     "r"(u[8 * q + 4]), "r"(u[8 * q + 5]), "r"(u[8 * q + 6]), "r"(u[8 * q + 7])
                     : "memory");
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q * 8 < cols)
        reinterpret_cast<uint4*>(dst)[q] =
            make_uint4(u[4 * q], u[4 * q + 1], u[4 * q + 2], u[4 * q + 3]);
  }
}
__device__ __forceinline__ void zero_cols(__nv_bfloat16* dst, int hd) {
  for (int c = 0; c < hd; c += 8) *reinterpret_cast<uint4*>(dst + c) = make_uint4(0, 0, 0, 0);
}

// ------------------------------------------------------- steps dealt out evenly
// Where whole units would leave many CTAs idle at the end, the gradient's steps
// (a unit's key or query tiles) are dealt out instead: CTA c of G takes steps
// [T c / G, T (c + 1) / G) of T. A unit that a border cuts is added up in pieces:
// every CTA stores the F32 sums of the first and the last unit of its range if it
// has them in part (slots 0 and 1), and a second kernel adds a unit's pieces in
// the order of the CTAs.
__device__ __forceinline__ int64_t border(int64_t total, int64_t c, int64_t ctas) {
  return total * c / ctas;
}
// 128 rows of HD F32 sums, two of them for each slot.
template <int HD>
__device__ __forceinline__ float* piece_rows(const TcArgs& a, int64_t cta, int slot, int t) {
  return a.piece + ((cta * 2 + slot) * 2 + t) * (int64_t)kRows * HD;
}
template <int HD>
__device__ __forceinline__ void store_piece32(float* row, const uint32_t (&v)[32]) {
#pragma unroll
  for (int q = 0; q < 8; ++q)
    reinterpret_cast<uint4*>(row)[q] = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
}
// The unit of steps [begin, begin + n) that border c cuts first: its pieces in
// order, as CTA * 2 + slot. Slot 0 of a CTA whose range begins in the unit, slot 1
// of the one whose range ends in it. One thread writes the list.
constexpr int kMostPieces = 1024;
__device__ __forceinline__ int list_pieces(int64_t total, int64_t ctas, int64_t c, int64_t begin,
                                           int64_t n, int* list) {
  int count = 0;
  for (int64_t i = c - 1; i < ctas && border(total, i, ctas) < begin + n; ++i) {
    if (border(total, i, ctas) == border(total, i + 1, ctas)) continue;  // nothing of its own
    list[count++] = (int)(i * 2 + (border(total, i, ctas) >= begin ? 0 : 1));
  }
  return count;
}
template <int HD>
__device__ __forceinline__ float4 sum_pieces(const TcArgs& a, const int* list, int count, int t,
                                             int row, int col) {
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = 0; i < count; ++i) {
    const float4 v = *reinterpret_cast<const float4*>(
        piece_rows<HD>(a, list[i] >> 1, list[i] & 1, t) + (int64_t)row * HD + col);
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  return s;
}
__device__ __forceinline__ void store_grad4(__nv_bfloat16* dst, float4 v, float mul) {
  const float x[4] = {v.x * mul, v.y * mul, v.z * mul, v.w * mul};
  store4(dst, x);
}

// 2^x of a pair on the FMA pipe, for x up to 8: x = n + f with n the nearest whole
// number (in the low bits of x + 1.5 2^23), a polynomial of degree 5 for 2^f on
// [-1/2, 1/2], n added to the exponent (the minimax polynomial by Remez exchange, whose
// relative error of 7.5e-8 its coefficients' rounding to F32 makes 1.55e-7, at most
// 2.2e-7 with the roundings of the F32 evaluation); 0 below 2^-126, as ex2.approx.ftz. A NaN becomes FLT_MAX (the bits of
// the canonical NaN, 0x7FFFFFFF, shifted and added to themselves), which the
// caller's sum has to turn back.
__device__ __forceinline__ void ex2_pair_fma(unsigned long long x, float& p0, float& p1) {
  const unsigned long long magic = f2_pack(12582912.f, 12582912.f);
  const unsigned long long t = f2_add(x, magic);
  const unsigned long long f = f2_sub(x, f2_sub(t, magic));
  auto c = [](float v) { return f2_pack(v, v); };
  unsigned long long y = f2_fma(c(0.0013276472454890609f), f, c(0.009675540961325169f));
  y = f2_fma(y, f, c(0.05550713092088699f));
  y = f2_fma(y, f, c(0.24022120237350464f));
  y = f2_fma(y, f, c(0.6931469440460205f));
  y = f2_fma(y, f, c(1.0000001192092896f));
  float x0, x1, t0, t1, y0, y1;
  f2_unpack(x, x0, x1);
  f2_unpack(t, t0, t1);
  f2_unpack(y, y0, y1);
  p0 = x0 < -126.f ? 0.f : __uint_as_float(__float_as_uint(t0) * 0x800000u + __float_as_uint(y0));
  p1 = x1 < -126.f ? 0.f : __uint_as_float(__float_as_uint(t1) * 0x800000u + __float_as_uint(y1));
}

// A sum of kv_len exponentials below 2^8 stays below 2^40: more is the FLT_MAX that
// ex2_pair_fma made of a NaN score.
__device__ __forceinline__ float nan_sum(float l) {
  return l > 1e30f ? __int_as_float(0x7fffffff) : l;
}

// A pair of (head, query tile) items that read the same key head: items 2p and
// 2p + 1 of the heads' query tiles in order.
struct PairUnit {
  int64_t b;
  int kvh, split, first;  // first item: (head in the group) * n_qt + query tile
  int items;
  int64_t len;
  int t0, n;  // first tile of the keys, number of tiles
};

// Head and query tile of a unit's tile t.
__device__ __forceinline__ int head_of(const TcArgs& a, const PairUnit& w, int t) {
  return w.kvh * a.g.group + (w.first + t) / a.n_qt;
}
__device__ __forceinline__ int tile_of(const TcArgs& a, const PairUnit& w, int t) {
  return (w.first + t) % a.n_qt;
}

template <int KT>
__device__ __forceinline__ PairUnit pair_of(const TcArgs& a, int b, int kvh, int split, int p) {
  const CrossGeom& g = a.g;
  PairUnit w;
  w.b = b;
  w.kvh = kvh;
  w.split = split;
  const int all = g.group * a.n_qt;
  w.first = 2 * p;
  w.items = 2 * p + 1 < all ? 2 : 1;
  w.len = cross_len(g, w.b);
  const int tiles = (int)((w.len + KT - 1) / KT);
  const int each = (tiles + a.n_split - 1) / a.n_split;
  w.t0 = w.split * each < tiles ? w.split * each : tiles;
  w.n = tiles - w.t0 < each ? tiles - w.t0 : each;
  return w;
}
// Unit numbers fit 32 bits (the host checks): a 64-bit division costs as much as
// half a tile.
template <int KT>
__device__ __forceinline__ PairUnit pair_unit(const TcArgs& a, const uint16_t* order, int u) {
  const uint32_t per_head = (uint32_t)(a.n_pairs * a.n_split);
  const uint32_t head = (uint32_t)u / per_head, x = (uint32_t)u % per_head;
  const uint32_t rank = head / (uint32_t)a.g.kv_heads, kvh = head % (uint32_t)a.g.kv_heads;
  return pair_of<KT>(a, sequence_of(a.g, order, (int)rank), (int)kvh, (int)(x / (uint32_t)a.n_pairs),
                     (int)(x % (uint32_t)a.n_pairs));
}

// =============================================================== forward
// Warps 0-3 turn S_0 into P_0, warps 4-7 S_1 into P_1. TMEM columns, head size
// 64: S_t at 128 t, O_t at 256 + 64 t, P_t (BF16 pairs, the A operand of P V) at
// 384 + 64 t, so S_t(j + 1) is computed as soon as S_t(j) has been read. Head
// size 128: S_t at 128 t, O_t at 256 + 128 t, and P_t takes the first half of
// S_t's columns: S_t(j + 1) follows P_t(j) V_j, and the other tile's softmax
// covers the wait. O_t is rescaled only when a row's maximum grows by more than
// 2^8 (the stale maximum is exact after the final division). P is rounded to BF16
// for P V, the row's sum adds the probabilities as they were before: the quotient is
// off by the rounding of each P, half a step.
template <int HD>
struct Fwd {
  static constexpr bool kOver = HD == 128;
  static constexpr int kBlocks = HD / 64;
  static constexpr int kTile = kBlocks * kBlk128;
  static constexpr int kQBufs = HD == 64 ? 2 : 1;
  static constexpr int kKs = HD == 64 ? 4 : 3, kVs = HD == 64 ? 4 : 2;
  static constexpr int kQ = 0;
  static constexpr int kK = kQBufs * 2 * kTile;
  static constexpr int kV = kK + kKs * kTile;
  static constexpr int kBar = kV + kVs * kTile;
  static constexpr int kBars = 2 * kQBufs + 2 * kKs + 2 * kVs + 10 + 1;
  static constexpr int kOrd = kBar + kBars * 8 + 8;
  static constexpr int kSmem = kOrd + 2 * kOrder + 1024;
  static_assert(kSmem <= 232448, "shared memory");
  __device__ static uint32_t tS(uint32_t t) { return t * 128; }
  __device__ static uint32_t tO(uint32_t t) { return 256 + t * HD; }
  __device__ static uint32_t tP(uint32_t t) { return kOver ? t * 128 : 384 + t * 64; }
};

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
cross_fwd_tc(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
             const __grid_constant__ CUtensorMap tmV, const __grid_constant__ TcArgs a) {
  using F = Fwd<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sp;
  const uint32_t base = align1024(smem_raw, &sp);
  auto sQ = [&](int qb, int t) { return base + F::kQ + (2 * qb + t) * F::kTile; };
  auto sK = [&](int st) { return base + F::kK + st * F::kTile; };
  auto sV = [&](int st) { return base + F::kV + st * F::kTile; };
  const uint32_t bars = base + F::kBar;
  auto q_full = [&](int i) { return bars + 8u * i; };
  auto q_empty = [&](int i) { return bars + 8u * (F::kQBufs + i); };
  const uint32_t kbars = bars + 16u * F::kQBufs;
  auto k_full = [&](int i) { return kbars + 8u * i; };
  auto k_empty = [&](int i) { return kbars + 8u * (F::kKs + i); };
  const uint32_t vbars = kbars + 16u * F::kKs;
  auto v_full = [&](int i) { return vbars + 8u * i; };
  auto v_empty = [&](int i) { return vbars + 8u * (F::kVs + i); };
  const uint32_t sbars = vbars + 16u * F::kVs;
  auto s_full = [&](int t) { return sbars + 8u * t; };
  auto s_free = [&](int t) { return sbars + 8u * (2 + t); };
  auto p_full = [&](int t) { return sbars + 8u * (4 + t); };
  auto p_half = [&](int t) { return sbars + 8u * (6 + t); };
  auto pv_done = [&](int t) { return sbars + 8u * (8 + t); };
  const uint32_t done_bar = sbars + 80u;
  const uint32_t tslot = bars + 8u * F::kBars;
  uint32_t* tslot_ptr = reinterpret_cast<uint32_t*>(sp + F::kBar + 8 * F::kBars);
  uint16_t* order = reinterpret_cast<uint16_t*>(sp + F::kOrd);

  const CrossGeom& g = a.g;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = (int)(a.n_pairs * a.n_split * g.kv_heads * g.batch);
  const int ctas = (int)gridDim.x, cta = (int)blockIdx.x;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&tmQ);
    prefetch_tensormap(&tmK);
    prefetch_tensormap(&tmV);
    for (int i = 0; i < F::kBars; ++i) {
      const uint32_t b = bars + 8u * i;
      const bool by_warps = b >= s_free(0) && b <= p_half(1);
      mbar_init(b, by_warps ? 4 : 1);
    }
    fence_barrier_init();
  }
  if (warp == kMmaWarp) tmem_alloc(tslot, 512);
  order_by_length(g, order);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tslot_ptr);

  if (warp == kTmaWarp) {
    if (elect_one()) {
      bool ok = true;
      int gk = 0;  // key tiles loaded so far
      int ru = 0;  // units that had keys
      for (int r = 0; ok; ++r) {
        const int u = snake(r, cta, ctas, units);
        if (u < 0) break;
        const PairUnit w = pair_unit<kRows>(a, order, u);
        if (w.n <= 0) continue;
        const int qb = ru % F::kQBufs;
        if (!mbar_wait(q_empty(qb), (uint32_t)(((ru / F::kQBufs) & 1) ^ 1), g.err)) break;
        mbar_expect_tx(q_full(qb), w.items * F::kTile);
        for (int t = 0; t < w.items; ++t)
          for (int c = 0; c < F::kBlocks; ++c)
            tma_load_4d(sQ(qb, t) + c * kBlk128, &tmQ, c * 64, tile_of(a, w, t) * kRows,
                        head_of(a, w, t) * a.qh, (int)w.b * a.qb, q_full(qb));
        for (int j = 0; j < w.n; ++j, ++gk) {
          const int ks = gk % F::kKs, vs = gk % F::kVs;
          const int row = (w.t0 + j) * kRows;
          if (!mbar_wait(k_empty(ks), (uint32_t)(((gk / F::kKs) & 1) ^ 1), g.err)) { ok = false; break; }
          mbar_expect_tx(k_full(ks), F::kTile);
          for (int c = 0; c < F::kBlocks; ++c)
            tma_load_4d(sK(ks) + c * kBlk128, &tmK, c * 64, row, w.kvh * a.kh, (int)w.b * a.kb,
                        k_full(ks));
          if (!mbar_wait(v_empty(vs), (uint32_t)(((gk / F::kVs) & 1) ^ 1), g.err)) { ok = false; break; }
          mbar_expect_tx(v_full(vs), F::kTile);
          for (int c = 0; c < F::kBlocks; ++c)
            tma_load_4d(sV(vs) + c * kBlk128, &tmV, c * 64, row, w.kvh * a.vh, (int)w.b * a.vb,
                        v_full(vs));
        }
        ++ru;
      }
      // every tile has been consumed before the producer leaves
      for (int i = gk; i < gk + F::kVs && ok; ++i)
        ok = mbar_wait(v_empty(i % F::kVs), (uint32_t)(((i / F::kVs) & 1) ^ 1), g.err);
    }
  } else if (warp == kMmaWarp) {
    if (elect_one()) {
      constexpr uint32_t idS = idesc_bf16_f32(kRows, kRows, 0, 0);
      constexpr uint32_t idO = idesc_bf16_f32(kRows, HD, 0, 1);
      const uint64_t dq0 = desc_k(sQ(0, 0)), dk0 = desc_k(sK(0)), dv0 = desc_mn(sV(0), kBlk128);
      bool ok = true;
      int ru = 0;
      // ring positions of the next key tile of S and of P V, and the parities of
      // their stages: counted up, so that nothing is divided per step
      int ks = 0, vs = 0;
      uint32_t kp = 0, vp = 0;
      uint32_t ns0 = 0, ns1 = 0, np0 = 0, np1 = 0;  // S_t, P_t V issued
      auto k_wait = [&]() {
        if (!mbar_wait(k_full(ks), kp, g.err)) return false;
        tc_fence_after();
        return true;
      };
      auto k_next = [&]() {  // both tiles' S have been issued
        mma_commit(k_empty(ks));
        if (++ks == F::kKs) ks = 0, kp ^= 1u;
      };
      auto issue_s = [&](auto tc, int qb) -> bool {
        constexpr int t = decltype(tc)::value;
        uint32_t& ns = t ? ns1 : ns0;
        if (!F::kOver && ns >= 1 && !mbar_wait(s_free(t), (ns - 1) & 1u, g.err)) return false;
        tc_fence_after();
        const uint64_t dq = desc_add(dq0, (uint32_t)(2 * qb + t) * F::kTile);
        const uint64_t dk = desc_add(dk0, (uint32_t)ks * F::kTile);
        const uint32_t d = tmem + F::tS(t);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          mma_bf16_ss(d, desc_add(dq, k_step(kk, kBlk128)), desc_add(dk, k_step(kk, kBlk128)), idS,
                      kk > 0 ? 1u : 0u);
        mma_commit(s_full(t));
        ++ns;
        return true;
      };
      auto issue_pv = [&](auto tc, uint32_t more) -> bool {
        constexpr int t = decltype(tc)::value;
        uint32_t& np = t ? np1 : np0;
        const uint64_t dv = desc_add(dv0, (uint32_t)vs * F::kTile);
        const uint32_t d = tmem + F::tO(t), p = tmem + F::tP(t);
        // the first 64 keys while the softmax is at the others
        if (!mbar_wait(p_half(t), np & 1u, g.err)) return false;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_bf16_ts(d, p + kk * 8, desc_add(dv, kk * 2048), idO, kk > 0 ? 1u : more);
        if (!mbar_wait(p_full(t), np & 1u, g.err)) return false;
        tc_fence_after();
#pragma unroll
        for (int kk = 4; kk < 8; ++kk)
          mma_bf16_ts(d, p + kk * 8, desc_add(dv, kk * 2048), idO, 1u);
        mma_commit(pv_done(t));
        ++np;
        return true;
      };
      using t0 = std::integral_constant<int, 0>;
      using t1 = std::integral_constant<int, 1>;
      int r = 0, u = snake(0, cta, ctas, units);
      PairUnit next{};
      if (u >= 0) next = pair_unit<kRows>(a, order, u);
      while (ok && u >= 0) {
        const PairUnit w = next;
        u = snake(++r, cta, ctas, units);
        if (w.n <= 0) {
          if (u >= 0) next = pair_unit<kRows>(a, order, u);
          continue;
        }
        const int qb = ru % F::kQBufs;
        const bool two = w.items > 1;
        ok = mbar_wait(q_full(qb), (uint32_t)((ru / F::kQBufs) & 1), g.err) && k_wait() &&
             issue_s(t0{}, qb) && (!two || issue_s(t1{}, qb));
        if (!ok) break;
        k_next();
        if (u >= 0) next = pair_unit<kRows>(a, order, u);  // while the first products run
        for (int j = 0; j < w.n; ++j) {
          const bool last = j + 1 == w.n;
          const uint32_t more = j > 0 ? 1u : 0u;
          ok = mbar_wait(v_full(vs), vp, g.err) && (last || k_wait());
          if (!ok) break;
          // head size 64: S_t(j + 1) as soon as S_t(j) has been read; 128: P_t(j)
          // lies in S_t's columns, so S_t(j + 1) goes behind P_t(j) V_j
          if constexpr (F::kOver) {
            ok = issue_pv(t0{}, more) && (last || issue_s(t0{}, qb)) &&
                 (!two || issue_pv(t1{}, more));
            if (!ok) break;
            mma_commit(v_empty(vs));
            if (two && !last) ok = issue_s(t1{}, qb);
          } else {
            ok = (last || issue_s(t0{}, qb)) && issue_pv(t0{}, more) &&
                 (!two || ((last || issue_s(t1{}, qb)) && issue_pv(t1{}, more)));
            if (!ok) break;
            mma_commit(v_empty(vs));
          }
          if (!ok) break;
          if (!last) k_next();
          if (++vs == F::kVs) vs = 0, vp ^= 1u;
        }
        if (!ok) break;
        ++ru;
        mma_commit(q_empty(qb));
      }
      mma_commit(done_bar);
      mbar_wait(done_bar, 0, g.err);
    }
  } else {
    const int t = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t srow = tmem + F::tS(t) + lanes;
    const uint32_t orow = tmem + F::tO(t) + lanes;
    const uint32_t prow = tmem + F::tP(t) + lanes;
    const float sl2 = scale_log2(g.scale);
    bool ok = true;
    int gs = 0;  // this warpgroup's steps so far
    int gk = 0;
    int r = 0;
    int u = snake(r, cta, ctas, units);
    PairUnit next{};
    if (u >= 0) next = pair_unit<kRows>(a, order, u);
    while (u >= 0) {
      const PairUnit w = next;
      u = snake(++r, cta, ctas, units);
      if (t >= w.items) {
        gk += w.n > 0 ? w.n : 0;
        if (u >= 0) next = pair_unit<kRows>(a, order, u);
        continue;
      }
      const int h = head_of(a, w, t);
      const int64_t qi = (int64_t)tile_of(a, w, t) * kRows + row;
      float m_run = -INFINITY, l_run = 0.f;
      for (int j = 0; j < w.n; ++j, ++gs, ++gk) {
        const int64_t left = w.len - (int64_t)(w.t0 + j) * kRows;
        const bool tail = left < kRows;
        const int lim = tail ? (int)left - 1 : kRows - 1;  // last key of the tile
        if (ok && !mbar_wait(s_full(t), (uint32_t)(gs & 1), g.err)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) continue;
        tc_fence_after();
        // The first 96 columns of the row stay in registers from the maximum to
        // the exponentials; the last 32 are read again (128 would not fit beside
        // the rest of the 168 a thread has).
        uint32_t v[3][32], w4[32];
        // -inf: no part in maximum or sum
        auto mask = [&](uint32_t(&x)[32], int c) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (c * 32 + e > lim) x[e] = 0xFF800000u;
        };
        tmem_ld32(srow + 96, w4);
#pragma unroll
        for (int c = 0; c < 3; ++c) tmem_ld32(srow + c * 32, v[c]);
        tmem_wait_ld();
        if (tail) {
          mask(w4, 3);
#pragma unroll
          for (int c = 0; c < 3; ++c) mask(v[c], c);
        }
        float mx8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) mx8[i] = __uint_as_float(w4[i]);
#pragma unroll
        for (int e = 8; e < 32; ++e) mx8[e & 7] = fmaxf(mx8[e & 7], __uint_as_float(w4[e]));
#pragma unroll
        for (int e = 0; e < 96; ++e)
          mx8[e & 7] = fmaxf(mx8[e & 7], __uint_as_float(v[e >> 5][e & 31]));
        const float mx = fmaxf(fmaxf(fmaxf(mx8[0], mx8[1]), fmaxf(mx8[2], mx8[3])),
                               fmaxf(fmaxf(mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
        const float m_new = fmaxf(m_run, mx * sl2);
        // The previous P V has read P_t and added into O_t (head size 128: S_t was
        // issued behind it, and is there).
        if constexpr (!F::kOver) {
          if (gs >= 1 && !mbar_wait(pv_done(t), (uint32_t)((gs - 1) & 1), g.err)) ok = false;
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) continue;
          tc_fence_after();
        }
        if (j == 0) {
          // scores of -inf alone: below any other, so that the first one to come rescales
          m_run = fmaxf(m_new, -FLT_MAX);
        } else if (__any_sync(0xffffffffu, m_new > m_run + kRescaleLog2)) {
          const float alpha = ex2_approx(m_run - m_new);
          m_run = m_new;
          l_run = nan_sum(l_run) * alpha;
#pragma unroll
          for (int c = 0; c < HD / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(orow + c * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st16(orow + c * 16, o);
          }
          tmem_wait_st();
        }
        // P = exp2(S scale log2(e) - m), two columns per instruction
        unsigned long long rs2[2] = {0ull, 0ull};
        const unsigned long long sl22 = f2_pack(sl2, sl2), nm2 = f2_pack(-m_run, -m_run);
        if (tail && t == 0) {  // P_0 V goes first: both tiles find the rows zeroed
          const int vs = gk % F::kVs;
          if (!mbar_wait(v_full(vs), (uint32_t)((gk / F::kVs) & 1), g.err)) ok = false;
          ok = __all_sync(0xffffffffu, ok);
          if (ok && row > lim) zero_row(sV(vs), row, F::kBlocks, kBlk128);
          fence_proxy_async_smem();
        }
        auto exp32 = [&](const uint32_t(&x)[32], int c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const unsigned long long z = f2_fma(
                f2_pack(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), sl22, nm2);
            float p0, p1;
            // A quarter of the exponentials run on the FMA pipe: the MUFU's 128 a row
            // are what the softmax waits for. (2048 queries, 4 x 32 heads, up to 4096
            // keys: none 298 us at head size 64 and 337 at 128, a quarter 279 and
            // 329, three eighths 284 and 334, half 314 and 355.)
            if (e % 4 == 3) {
              ex2_pair_fma(z, p0, p1);
            } else {
              float x0, x1;
              f2_unpack(z, x0, x1);
              p0 = ex2_approx(x0);
              p1 = ex2_approx(x1);
            }
            rs2[e & 1] = f2_add(rs2[e & 1], f2_pack(p0, p1));
            pk[e] = pack_bf16(p0, p1);
          }
          tmem_st16(prow + c * 16, pk);
        };
        auto arrive = [&](uint32_t bar) {
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (ok && lane == 0) mbar_arrive(bar);
        };
        exp32(v[0], 0);
        exp32(v[1], 1);
        arrive(p_half(t));
        tmem_ld32(srow + 96, w4);
        exp32(v[2], 2);
        tmem_wait_ld();
        if (!F::kOver) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(s_free(t));
        }
        if (tail) mask(w4, 3);
        exp32(w4, 3);
        arrive(p_full(t));
        float a0, a1, b0, b1;
        f2_unpack(rs2[0], a0, a1);
        f2_unpack(rs2[1], b0, b1);
        l_run += (a0 + a1) + (b0 + b1);
      }
      if (u >= 0) next = pair_unit<kRows>(a, order, u);  // while the last product runs
      if (ok && w.n > 0 && !mbar_wait(pv_done(t), (uint32_t)((gs - 1) & 1), g.err)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) continue;
      tc_fence_after();
      l_run = nan_sum(l_run);
      const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;  // no keys: a zero row
      const float lse = l_run == 0.f ? -INFINITY : m_run * kLn2 + logf(l_run);
      const int64_t at = (w.b * g.heads + h) * g.q_len + qi;
      const bool in = qi < g.q_len;
      __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.o) + w.b * g.os[0] + h * g.os[1] +
                           qi * g.os[2];
      const int64_t pat = w.split * g.batch * g.heads * g.q_len + at;
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t v[32];
        if (w.n > 0) {
          tmem_ld32(orow + c * 32, v);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0u;
        }
        if (!in || c * 32 >= g.hd) continue;
        if (a.n_split == 1) {
          store_cols32(dst + c * 32, v, inv, g.hd - c * 32);
        } else {
          float4* pd = reinterpret_cast<float4*>(a.part + pat * g.hd + c * 32);
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (c * 32 + q * 4 < g.hd)
              pd[q] = make_float4(__uint_as_float(v[4 * q]) * inv, __uint_as_float(v[4 * q + 1]) * inv,
                                  __uint_as_float(v[4 * q + 2]) * inv,
                                  __uint_as_float(v[4 * q + 3]) * inv);
        }
      }
      if (in) {
        if (a.n_split > 1) a.part_lse[pat] = lse;
        else if (a.lse != nullptr) a.lse[at] = lse;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// =========================================================== rows of the gradient
// nlse = -lse log2(e), delta = rowsum(dO O), rows padded to a multiple of 64 with
// (-inf, 0): the exponential of a row that is not there, or that had no
// probabilities, is 0. A CTA per 64 rows, eight threads a row, four rows a thread, whose
// reads are all on their way at once: 7 us for the 17 MB of 8 x 16 heads, 512 rows of 64
// (one row a thread 8), 14 us for the 67 MB of 2 x 32 heads, 2048 rows of 128 (16).
__global__ void __launch_bounds__(128)
cross_rows(const __nv_bfloat16* __restrict__ o, const __nv_bfloat16* __restrict__ d_o,
           const float* __restrict__ lse, float* __restrict__ nlse, float* __restrict__ delta,
           const CrossGeom g, int q_pad) {
  constexpr int kEach = 4;
  let_next_launch_begin();
  const uint32_t per_head = (uint32_t)q_pad / 64, bh = blockIdx.x / per_head;
  const uint32_t b = bh / (uint32_t)g.heads, h = bh % (uint32_t)g.heads;
  const int64_t q0 = (int64_t)(blockIdx.x % per_head) * 64 + (threadIdx.x >> 3);
  const int part = threadIdx.x & 7;
  const __nv_bfloat16* po = o + b * g.os[0] + h * g.os[1] + part * 8;
  const __nv_bfloat16* pd = d_o + b * g.dos[0] + h * g.dos[1] + part * 8;
  uint4 x[kEach][2], y[kEach][2];
#pragma unroll
  for (int u = 0; u < kEach; ++u)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int64_t q = q0 + 16 * u;
      x[u][c] = y[u][c] = make_uint4(0u, 0u, 0u, 0u);
      if (q < g.q_len && part * 8 + 64 * c < g.hd) {
        x[u][c] = *reinterpret_cast<const uint4*>(po + q * g.os[2] + 64 * c);
        y[u][c] = *reinterpret_cast<const uint4*>(pd + q * g.dos[2] + 64 * c);
      }
    }
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    const int64_t q = q0 + 16 * u;
    float acc = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint32_t xs[4] = {x[u][c].x, x[u][c].y, x[u][c].z, x[u][c].w};
      const uint32_t ys[4] = {y[u][c].x, y[u][c].y, y[u][c].z, y[u][c].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc = fmaf(__uint_as_float(xs[e] << 16), __uint_as_float(ys[e] << 16), acc);
        acc = fmaf(__uint_as_float(xs[e] & 0xFFFF0000u), __uint_as_float(ys[e] & 0xFFFF0000u), acc);
      }
    }
#pragma unroll
    for (int w = 4; w > 0; w >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, w);
    if (part != 0) continue;
    float l = -INFINITY;
    if (q < g.q_len) {
      const float v = lse[(int64_t)bh * g.q_len + q];
      l = v == -INFINITY ? -INFINITY : -v * kLog2e;
    }
    nlse[(int64_t)bh * q_pad + q] = l;
    delta[(int64_t)bh * q_pad + q] = acc;
  }
}

// P of 32 columns of a row in place of S, two columns per instruction; nl: the
// -lse log2(e) of a column pair.
template <typename NL>
__device__ __forceinline__ void probs32(uint32_t (&v)[32], unsigned long long sl22, NL nl) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    float x0, x1;
    f2_unpack(f2_fma(f2_pack(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), sl22, nl(e)),
              x0, x1);
    v[2 * e] = __float_as_uint(ex2_approx(x0));
    v[2 * e + 1] = __float_as_uint(ex2_approx(x1));
  }
}
// dS = P (dP - delta) of 32 columns as BF16 pairs; dl: the delta of a column pair.
template <typename DL>
__device__ __forceinline__ void grads32(const uint32_t (&p)[32], const uint32_t (&vd)[32], DL dl,
                                        uint32_t (&pd)[16]) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    float d0, d1;
    f2_unpack(f2_mul(f2_pack(__uint_as_float(p[2 * e]), __uint_as_float(p[2 * e + 1])),
                     f2_sub(f2_pack(__uint_as_float(vd[2 * e]), __uint_as_float(vd[2 * e + 1])),
                            dl(e))), d0, d1);
    pd[e] = pack_bf16(d0, d1);
  }
}

// What the BF16 pairs of 32 columns leave of their F32 values, as BF16 pairs.
__device__ __forceinline__ void rest16(const uint32_t (&x)[32], const uint32_t (&hi)[16],
                                       uint32_t (&lo)[16]) {
#pragma unroll
  for (int e = 0; e < 16; ++e)
    lo[e] = pack_bf16(__uint_as_float(x[2 * e]) - __uint_as_float(hi[e] << 16),
                      __uint_as_float(x[2 * e + 1]) - __uint_as_float(hi[e] & 0xFFFF0000u));
}
// dS of 32 columns as F32, in place of dP.
template <typename DL>
__device__ __forceinline__ void grads32_f32(const uint32_t (&p)[32], uint32_t (&vd)[32], DL dl) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    float d0, d1;
    f2_unpack(f2_mul(f2_pack(__uint_as_float(p[2 * e]), __uint_as_float(p[2 * e + 1])),
                     f2_sub(f2_pack(__uint_as_float(vd[2 * e]), __uint_as_float(vd[2 * e + 1])),
                            dl(e))), d0, d1);
    vd[2 * e] = __float_as_uint(d0);
    vd[2 * e + 1] = __float_as_uint(d1);
  }
}
__device__ __forceinline__ void pack32(const uint32_t (&x)[32], uint32_t (&hi)[16]) {
#pragma unroll
  for (int e = 0; e < 16; ++e)
    hi[e] = pack_bf16(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]));
}

// =================================================================== dQ
// As the forward kernel, over 64-key tiles: S_t, dP_t = dO_t V_j^T; dS_t as BF16
// pairs in S_t's columns is the A operand of dQ_t += dS_t K_j (SPLIT: in two terms, as
// in cross_dkdv_tc). TMEM columns of
// tile t from 256 t: S, dP, dQ.
constexpr int kDealt = kOrder / 2;  // entries of a table of steps, in the place of the order

// Steps of the pairs of all sequences: first[b] of the sequences before b. One
// warp fills the table; without lengths every sequence has as many. (The host
// deals out fewer than 2^31 steps.)
__device__ __forceinline__ void step_table(const TcArgs& a, int keys, int* first) {
  const CrossGeom& g = a.g;
  const int lane = threadIdx.x & 31;
  const int pairs = (int)(a.n_pairs * g.kv_heads), batch = (int)g.batch;
  int sum = 0;
  for (int i0 = 0; i0 < batch; i0 += 32) {
    const int i = i0 + lane;
    const int n = i < batch ? ((int)cross_len(g, i) + keys - 1) / keys * pairs : 0;
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    if (i < batch) first[i] = sum + inc - n;
    sum += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) first[batch] = sum;
}

// Where step s of all lies: its sequence, the pair, the key tile in the pair.
struct StepAt {
  int b, pair, n, j;  // n: key tiles of the sequence
};
__device__ __forceinline__ StepAt step_at(const TcArgs& a, int keys, const int* first, int s) {
  const CrossGeom& g = a.g;
  StepAt x;
  uint32_t rest;
  if (g.lens != nullptr) {
    int lo = 0, hi = (int)g.batch;  // first[lo] <= s < first[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= s) lo = mid;
      else hi = mid;
    }
    x.b = lo;
    x.n = ((int)cross_len(g, lo) + keys - 1) / keys;
    rest = (uint32_t)(s - first[lo]);
  } else {
    x.n = ((int)g.kv_len + keys - 1) / keys;
    const uint32_t per = (uint32_t)(x.n * a.n_pairs * g.kv_heads);
    x.b = (int)((uint32_t)s / per);
    rest = (uint32_t)s % per;
  }
  x.pair = (int)(rest / (uint32_t)x.n);
  x.j = (int)(rest % (uint32_t)x.n);
  return x;
}
__device__ __forceinline__ int steps_of_all(const TcArgs& a, int keys, const int* first) {
  const CrossGeom& g = a.g;
  return g.lens != nullptr
             ? first[g.batch]
             : (int)((g.kv_len + keys - 1) / keys * a.n_pairs * g.kv_heads * g.batch);
}

// A CTA's way through its work: whole units in a snake, or its range of steps.
struct DqWalk {
  int r = 0, s = 0, end = 0;
};
struct DqUnit : PairUnit {
  int j0, j1, slot;  // key tiles [j0, j1); slot of the partial sums, -1: the unit is whole
};
template <int KT>
__device__ __forceinline__ bool dq_next(const TcArgs& a, const uint16_t* order, const int* first,
                                        int total, DqWalk& k, DqUnit& w) {
  const CrossGeom& g = a.g;
  if (a.piece == nullptr) {
    const int u =
        snake(k.r, (int)blockIdx.x, (int)gridDim.x, (int)(a.n_pairs * g.kv_heads * g.batch));
    if (u < 0) return false;
    ++k.r;
    static_cast<PairUnit&>(w) = pair_unit<KT>(a, order, u);
    w.j0 = 0;
    w.j1 = w.n;
    w.slot = -1;
    return true;
  }
  bool first_piece = false;
  if (k.r == 0) {
    k.r = 1;
    k.s = (int)border(total, blockIdx.x, gridDim.x);
    k.end = (int)border(total, blockIdx.x + 1, gridDim.x);
    first_piece = true;
  }
  if (k.s >= k.end) return false;
  const StepAt x = step_at(a, KT, first, k.s);
  static_cast<PairUnit&>(w) = pair_of<KT>(a, x.b, x.pair / a.n_pairs, 0, x.pair % a.n_pairs);
  w.j0 = x.j;
  const int stop = x.j + (k.end - k.s);
  w.j1 = stop < x.n ? stop : x.n;
  w.slot = w.j1 - w.j0 == x.n ? -1 : first_piece ? 0 : 1;
  k.s += w.j1 - w.j0;
  return true;
}

template <int HD>
struct Dq {
  static constexpr int kKeys = 64;
  static constexpr int kBlocks = HD / 64;
  static constexpr int kTile = kBlocks * kBlk128;   // Q, dO
  static constexpr int kKv = kBlocks * kBlk64;      // K, V
  static constexpr int kStages = HD == 64 ? 6 : 3;
  static constexpr int kQ = 0;                      // [t][Q, dO]
  static constexpr int kRing = 4 * kTile;           // [stage][K, V]
  static constexpr int kBar = kRing + kStages * 2 * kKv;
  static constexpr int kBars = 2 + 2 * kStages + 8 + 1;
  static constexpr int kOrd = kBar + kBars * 8 + 8;
  static constexpr int kSmem = kOrd + 2 * kOrder + 1024;
  static_assert(kSmem <= 232448, "shared memory");
};

template <int HD, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
cross_dq_tc(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmG,
            const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
            const __grid_constant__ TcArgs a) {
  using F = Dq<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sp;
  const uint32_t base = align1024(smem_raw, &sp);
  auto sQ = [&](int t) { return base + F::kQ + 2 * t * F::kTile; };
  auto sG = [&](int t) { return base + F::kQ + (2 * t + 1) * F::kTile; };
  auto sK = [&](int st) { return base + F::kRing + 2 * st * F::kKv; };
  auto sV = [&](int st) { return base + F::kRing + (2 * st + 1) * F::kKv; };
  const uint32_t bars = base + F::kBar;
  const uint32_t q_full = bars, q_empty = bars + 8;
  auto kv_full = [&](int i) { return bars + 8u * (2 + i); };
  auto kv_empty = [&](int i) { return bars + 8u * (2 + F::kStages + i); };
  const uint32_t sbars = bars + 8u * (2 + 2 * F::kStages);
  auto s_full = [&](int t) { return sbars + 8u * t; };
  auto ds_full = [&](int t) { return sbars + 8u * (2 + t); };
  auto dq_done = [&](int t) { return sbars + 8u * (4 + t); };
  auto dp_full = [&](int t) { return sbars + 8u * (6 + t); };
  const uint32_t done_bar = sbars + 64u;
  const uint32_t tslot = bars + 8u * F::kBars;
  uint32_t* tslot_ptr = reinterpret_cast<uint32_t*>(sp + F::kBar + 8 * F::kBars);
  // the order of the sequences, or the table of their steps
  uint16_t* order = reinterpret_cast<uint16_t*>(sp + F::kOrd);
  int* first = reinterpret_cast<int*>(sp + F::kOrd);

  const CrossGeom& g = a.g;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctas = (int)gridDim.x, cta = (int)blockIdx.x;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&tmQ);
    prefetch_tensormap(&tmG);
    prefetch_tensormap(&tmK);
    prefetch_tensormap(&tmV);
    for (int i = 0; i < F::kBars; ++i) {
      const uint32_t b = bars + 8u * i;
      mbar_init(b, b == ds_full(0) || b == ds_full(1) ? 4 : 1);
    }
    fence_barrier_init();
  }
  if (warp == kMmaWarp) tmem_alloc(tslot, 512);
  if (a.piece == nullptr) order_by_length(g, order);
  else if (g.lens != nullptr && warp == 0) step_table(a, F::kKeys, first);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tslot_ptr);
  const int total = a.piece == nullptr ? 0 : steps_of_all(a, F::kKeys, first);
  auto tS = [&](int t) { return tmem + 256u * t; };
  auto tDp = [&](int t) { return tmem + 256u * t + 64u; };
  auto tDq = [&](int t) { return tmem + 256u * t + 128u; };

  if (warp == kTmaWarp) {
    if (elect_one()) {
      bool ok = true;
      int gk = 0, ru = 0;
      DqWalk walk;
      DqUnit w;
      while (ok && dq_next<F::kKeys>(a, order, first, total, walk, w)) {
        if (w.n <= 0) continue;
        if (!mbar_wait(q_empty, (uint32_t)((ru & 1) ^ 1), g.err)) break;
        mbar_expect_tx(q_full, w.items * 2 * F::kTile);
        for (int t = 0; t < w.items; ++t)
          for (int c = 0; c < F::kBlocks; ++c) {
            const int row = tile_of(a, w, t) * kRows, h = head_of(a, w, t);
            tma_load_4d(sQ(t) + c * kBlk128, &tmQ, c * 64, row, h * a.qh, (int)w.b * a.qb, q_full);
            tma_load_4d(sG(t) + c * kBlk128, &tmG, c * 64, row, h * a.dh, (int)w.b * a.db, q_full);
          }
        for (int j = w.j0; j < w.j1; ++j, ++gk) {
          const int st = gk % F::kStages, row = j * F::kKeys;
          if (!mbar_wait(kv_empty(st), (uint32_t)(((gk / F::kStages) & 1) ^ 1), g.err)) {
            ok = false;
            break;
          }
          mbar_expect_tx(kv_full(st), 2 * F::kKv);
          for (int c = 0; c < F::kBlocks; ++c) {
            tma_load_4d(sK(st) + c * kBlk64, &tmK, c * 64, row, w.kvh * a.kh, (int)w.b * a.kb,
                        kv_full(st));
            tma_load_4d(sV(st) + c * kBlk64, &tmV, c * 64, row, w.kvh * a.vh, (int)w.b * a.vb,
                        kv_full(st));
          }
        }
        ++ru;
      }
      for (int i = gk; i < gk + F::kStages && ok; ++i)
        ok = mbar_wait(kv_empty(i % F::kStages), (uint32_t)(((i / F::kStages) & 1) ^ 1), g.err);
    }
  } else if (warp == kMmaWarp) {
    if (elect_one()) {
      constexpr uint32_t idS = idesc_bf16_f32(kRows, F::kKeys, 0, 0);
      constexpr uint32_t idQ = idesc_bf16_f32(kRows, HD, 0, 1);
      bool ok = true;
      int ru = 0;
      const uint64_t dq0 = desc_k(sQ(0)), dg0 = desc_k(sG(0)), dk0 = desc_k(sK(0)),
                     dv0 = desc_k(sV(0)), dkm0 = desc_mn(sK(0), kBlk64);
      int sst = 0, gst = 0;      // ring stages of the next S / dP and of the next dQ
      uint32_t sph = 0;
      uint32_t nd0 = 0, nd1 = 0;  // dS_t used
      auto kv_wait = [&]() {
        if (!mbar_wait(kv_full(sst), sph, g.err)) return false;
        tc_fence_after();
        return true;
      };
      auto kv_next = [&]() {
        if (++sst == F::kStages) sst = 0, sph ^= 1u;
      };
      auto issue_s = [&](auto tc) {
        constexpr int t = decltype(tc)::value;
        const uint64_t dk = desc_add(dk0, (uint32_t)sst * 2 * F::kKv);
        const uint64_t dv = desc_add(dv0, (uint32_t)sst * 2 * F::kKv);
        constexpr uint32_t at = (uint32_t)t * 2 * F::kTile;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          mma_bf16_ss(tS(t), desc_add(dq0, at + k_step(kk, kBlk128)), desc_add(dk, k_step(kk, kBlk64)),
                      idS, kk > 0 ? 1u : 0u);
        mma_commit(s_full(t));
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          mma_bf16_ss(tDp(t), desc_add(dg0, at + k_step(kk, kBlk128)),
                      desc_add(dv, k_step(kk, kBlk64)), idS, kk > 0 ? 1u : 0u);
        mma_commit(dp_full(t));
      };
      auto issue_dq = [&](auto tc, uint32_t more) -> bool {
        constexpr int t = decltype(tc)::value;
        uint32_t& nd = t ? nd1 : nd0;
        if (!mbar_wait(ds_full(t), nd & 1u, g.err)) return false;
        ++nd;
        tc_fence_after();
        const uint64_t dk = desc_add(dkm0, (uint32_t)gst * 2 * F::kKv);
#pragma unroll
        for (int kk = 0; kk < F::kKeys / 16; ++kk)
          mma_bf16_ts(tDq(t), tS(t) + kk * 8, desc_add(dk, kk * 2048), idQ, kk > 0 ? 1u : more);
        if constexpr (SPLIT) {
#pragma unroll
          for (int kk = 0; kk < F::kKeys / 16; ++kk)
            mma_bf16_ts(tDq(t), tS(t) + 32u + kk * 8, desc_add(dk, kk * 2048), idQ, 1u);
        }
        return true;
      };
      using t0 = std::integral_constant<int, 0>;
      using t1 = std::integral_constant<int, 1>;
      DqWalk walk;
      DqUnit next;
      bool have = dq_next<F::kKeys>(a, order, first, total, walk, next);
      while (ok && have) {
        const DqUnit w = next;
        if (w.n <= 0) {
          have = dq_next<F::kKeys>(a, order, first, total, walk, next);
          continue;
        }
        const bool two = w.items > 1;
        ok = mbar_wait(q_full, (uint32_t)(ru & 1), g.err) && kv_wait();
        if (!ok) break;
        issue_s(t0{});
        if (two) issue_s(t1{});
        kv_next();
        have = dq_next<F::kKeys>(a, order, first, total, walk, next);  // while they run
        for (int j = w.j0; j < w.j1; ++j) {
          const bool last = j + 1 == w.j1;
          const uint32_t more = j > w.j0 ? 1u : 0u;
          ok = (last || kv_wait()) && issue_dq(t0{}, more);
          if (!ok) break;
          if (last) mma_commit(dq_done(0));
          else issue_s(t0{});
          if (two) {
            ok = issue_dq(t1{}, more);
            if (!ok) break;
          }
          mma_commit(kv_empty(gst));
          if (two) {
            if (last) mma_commit(dq_done(1));
            else issue_s(t1{});
          }
          if (!last) kv_next();
          if (++gst == F::kStages) gst = 0;
        }
        if (!ok) break;
        ++ru;
        mma_commit(q_empty);
      }
      mma_commit(done_bar);
      mbar_wait(done_bar, 0, g.err);
    }
  } else {
    wait_for_launch_before();  // for the row terms
    if (a.piece == nullptr) let_next_launch_begin();
    const int t = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const float sl2 = scale_log2(g.scale);
    const unsigned long long sl22 = f2_pack(sl2, sl2);
    bool ok = true;
    int gs = 0, gk = 0, gu = 0;
    DqWalk walk;
    DqUnit next;
    bool have = dq_next<F::kKeys>(a, order, first, total, walk, next);
    while (have) {
      const DqUnit w = next;
      if (t >= w.items) {
        gk += w.j1 > w.j0 ? w.j1 - w.j0 : 0;
        have = dq_next<F::kKeys>(a, order, first, total, walk, next);
        continue;
      }
      const int h = head_of(a, w, t);
      const int64_t qi = (int64_t)tile_of(a, w, t) * kRows + row;
      const bool in = qi < g.q_len;
      const int64_t at = (w.b * g.heads + h) * a.q_pad + qi;
      const float nl = in ? a.nlse[at] : -INFINITY, dl = in ? a.delta[at] : 0.f;
      const unsigned long long nl2 = f2_pack(nl, nl);
      unsigned long long dl2 = f2_pack(dl, dl);
      for (int j = w.j0; j < w.j1; ++j, ++gs, ++gk) {
        const int64_t left = w.len - (int64_t)j * F::kKeys;
        const bool tail = left < F::kKeys;
        const int lim = tail ? (int)left - 1 : F::kKeys - 1;
        if (ok && !mbar_wait(s_full(t), (uint32_t)(gs & 1), g.err)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) continue;
        tc_fence_after();
        uint32_t vs[2][32];
        tmem_ld32(tS(t) + lanes, vs[0]);
        tmem_ld32(tS(t) + lanes + 32, vs[1]);
        tmem_wait_ld();
        // P while dP is being computed
#pragma unroll
        for (int c = 0; c < 2; ++c) probs32(vs[c], sl22, [&](int) { return nl2; });
        if (!mbar_wait(dp_full(t), (uint32_t)(gs & 1), g.err)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) continue;
        tc_fence_after();
        if (w.n == 1) {
          // All keys of the row are here: delta = sum P dP without the rounding of
          // the stored O, which a few keys do not average out. dK reads it too.
          float sum = 0.f;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t vd[32];
            tmem_ld32(tDp(t) + lanes + 32 * c, vd);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (32 * c + e <= lim)
                sum = fmaf(__uint_as_float(vs[c][e]), __uint_as_float(vd[e]), sum);
          }
          dl2 = f2_pack(sum, sum);
          if (in) a.delta[at] = sum;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t vd[32], pd[16];
          tmem_ld32(tDp(t) + lanes + 32 * c, vd);
          tmem_wait_ld();
          auto mask = [&](uint32_t(&x)[16]) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              if (32 * c + 2 * e > lim) x[e] &= 0xFFFF0000u;
              if (32 * c + 2 * e + 1 > lim) x[e] &= 0x0000FFFFu;
            }
          };
          if constexpr (SPLIT) {
            uint32_t pl[16];
            grads32_f32(vs[c], vd, [&](int) { return dl2; });
            pack32(vd, pd);
            rest16(vd, pd, pl);
            if (tail) mask(pl);
            tmem_st16(tS(t) + lanes + 32 + 16 * c, pl);
          } else {
            grads32(vs[c], vd, [&](int) { return dl2; }, pd);
          }
          if (tail) mask(pd);
          tmem_st16(tS(t) + lanes + 16 * c, pd);  // S_t is in registers
        }
        if (tail && t == 0 && row < F::kKeys) {  // warps 0 and 1
          const int st = gk % F::kStages;
          if (!mbar_wait(kv_full(st), (uint32_t)((gk / F::kStages) & 1), g.err)) ok = false;
          ok = __all_sync(0xffffffffu, ok);
          if (ok && row > lim) zero_row(sK(st), row, F::kBlocks, kBlk64);
          fence_proxy_async_smem();
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(ds_full(t));
      }
      __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.dq) + w.b * g.dqs[0] + h * g.dqs[1] +
                           qi * g.dqs[2];
      have = dq_next<F::kKeys>(a, order, first, total, walk, next);  // while the last products run
      if (w.n <= 0) {
        if (in) zero_cols(dst, g.hd);
        continue;
      }
      if (ok && !mbar_wait(dq_done(t), (uint32_t)(gu & 1), g.err)) ok = false;
      ++gu;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) continue;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t v[32];
        tmem_ld32(tDq(t) + lanes + c * 32, v);
        tmem_wait_ld();
        if (w.slot >= 0)
          store_piece32<HD>(piece_rows<HD>(a, cta, w.slot, t) + (int64_t)row * HD + c * 32, v);
        else if (in && c * 32 < g.hd)
          store_cols32(dst + c * 32, v, g.scale, g.hd - c * 32);
      }
    }
    // sequences without keys have no steps
    if (a.piece != nullptr && g.lens != nullptr) {
      const int64_t rows = (int64_t)g.heads * g.q_len;
      for (int64_t b = 0; b < g.batch; ++b) {
        if (first[b + 1] != first[b]) continue;
        for (int64_t i = (int64_t)cta * 256 + threadIdx.x; i < rows; i += (int64_t)ctas * 256)
          zero_cols(static_cast<__nv_bfloat16*>(a.dq) + b * g.dqs[0] + i / g.q_len * g.dqs[1] +
                        i % g.q_len * g.dqs[2], g.hd);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// dQ of the pairs that a border of the steps cuts: a CTA per border and eighth of
// the pair's 256 rows.
template <int HD>
__global__ void __launch_bounds__(256)
cross_dq_join(const __grid_constant__ TcArgs a, int ctas) {
  __shared__ int first[kDealt];
  __shared__ int list[kMostPieces], count;
  wait_for_launch_before();
  const CrossGeom& g = a.g;
  constexpr int kKeys = Dq<HD>::kKeys;
  if (g.lens != nullptr && threadIdx.x < 32) step_table(a, kKeys, first);
  __syncthreads();
  const int64_t total = steps_of_all(a, kKeys, first), c = (int64_t)blockIdx.x + 1;
  const int64_t s = border(total, c, ctas);
  if (s >= total) return;
  const StepAt x = step_at(a, kKeys, first, (int)s);
  const int64_t begin = s - x.j;
  // the unit begins here, or an earlier border has it
  if (x.j == 0 || border(total, c - 1, ctas) > begin) return;
  const PairUnit w = pair_of<kKeys>(a, x.b, x.pair / a.n_pairs, 0, x.pair % a.n_pairs);
  if (threadIdx.x == 0) count = list_pieces(total, ctas, c, begin, x.n, list);
  __syncthreads();
  constexpr int kVec = HD / 4;
  const int t = (int)blockIdx.y / 4;  // four CTAs a tile
  if (t >= w.items) return;
  const int h = head_of(a, w, t);
  const int64_t q0 = (int64_t)tile_of(a, w, t) * kRows;
  __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.dq) + w.b * g.dqs[0] + h * g.dqs[1];
#pragma unroll 2
  for (int i = threadIdx.x; i < 32 * kVec; i += 256) {
    const int row = (int)(blockIdx.y % 4) * 32 + i / kVec, col = i % kVec * 4;
    if (col >= g.hd || q0 + row >= g.q_len) continue;
    store_grad4(dst + (q0 + row) * g.dqs[2] + col, sum_pieces<HD>(a, list, count, t, row, col),
                g.scale);
  }
}

// ================================================================ dK and dV
// A unit is a 128-key tile of a key head; its steps are the 64-query tiles of
// all query heads that share it. Steps alternate between two score buffers and
// the two warpgroups: S^T = K Q^T, dP^T = V dO^T (thread = key row); P^T and
// dS^T as BF16 pairs in the same columns are the A operands of dV += P^T dO and
// dK += dS^T Q (SPLIT: what the pairs left of the F32 values, as pairs in the upper
// half of the columns, is a second A operand). TMEM columns of buffer t from 128 t: S^T, dP^T; then dV, dK.
// Nothing is masked: a row of a key behind the length only reaches its own
// output row, which is stored as zeros, and the terms of a query row behind
// q_len make its probabilities 0.
//
// Whole units go round in a snake as far as they fill all CTAs; the rest of them
// is dealt out by steps.
struct KvUnit {
  int64_t b, len;
  int kvh, kt;
  int i0, i1, slot;  // steps [i0, i1); slot of the partial sums, -1: the unit is whole
};
struct KvWalk {
  int r = 0, s = -1, end = 0;
};
// first[i]: key tiles of the sequences before i, of one key head.
__device__ __forceinline__ bool kv_table(const CrossGeom& g) {
  return g.lens != nullptr && g.batch < kOrder;
}
__device__ __forceinline__ void tile_table(const CrossGeom& g, int* first) {
  const int lane = threadIdx.x & 31, batch = (int)g.batch;
  int sum = 0;
  for (int i0 = 0; i0 < batch; i0 += 32) {
    const int i = i0 + lane;
    const int n = i < batch ? (int)((cross_len(g, i) + kRows - 1) / kRows) : 0;
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    if (i < batch) first[i] = sum + inc - n;
    sum += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) first[batch] = sum;
}
// Unit u: sequences outermost, then key heads, then tiles, so that tiles that run
// at the same time read the same queries. With a table the units are exactly the
// tiles that have keys; without one every tile is a unit.
__device__ __forceinline__ KvUnit kv_unit(const CrossGeom& g, const int* first, int u, int n_it) {
  KvUnit w;
  const uint32_t heads = (uint32_t)g.kv_heads;
  uint32_t tiles, rest;
  if (kv_table(g)) {
    int lo = 0, hi = (int)g.batch;  // first[lo] * heads <= u < first[hi] * heads
    const int x = (int)((uint32_t)u / heads);
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= x) lo = mid;
      else hi = mid;
    }
    w.b = lo;
    tiles = (uint32_t)(first[lo + 1] - first[lo]);
    rest = (uint32_t)u - (uint32_t)first[lo] * heads;
  } else {
    tiles = (uint32_t)((g.kv_len + kRows - 1) / kRows);
    w.b = (uint32_t)u / (tiles * heads);
    rest = (uint32_t)u % (tiles * heads);
  }
  w.kvh = (int)(rest / tiles);
  w.kt = (int)(rest % tiles);
  w.len = cross_len(g, w.b);
  w.i0 = 0;
  w.i1 = (int64_t)w.kt * kRows < w.len ? n_it : 0;
  w.slot = -1;
  return w;
}
__device__ __forceinline__ int kv_units(const CrossGeom& g, const int* first) {
  return (int)((kv_table(g) ? first[g.batch] : (g.kv_len + kRows - 1) / kRows * g.batch) * g.kv_heads);
}
// Units that go round whole; the others' steps are dealt out.
__device__ __forceinline__ int kv_whole(const TcArgs& a, int units, int ctas) {
  return a.piece == nullptr ? units : units / ctas * ctas;
}
__device__ __forceinline__ bool kv_next(const TcArgs& a, const int* first, int units, int n_it,
                                        KvWalk& k, KvUnit& w) {
  const int ctas = (int)gridDim.x, cta = (int)blockIdx.x;
  const int whole = kv_whole(a, units, ctas);
  bool first_piece = false;
  if (k.s < 0) {
    const int u = snake(k.r, cta, ctas, whole);
    if (u >= 0) {
      ++k.r;
      w = kv_unit(a.g, first, u, n_it);
      return true;
    }
    const int64_t total = (int64_t)(units - whole) * n_it;
    k.s = (int)border(total, cta, ctas);
    k.end = (int)border(total, cta + 1, ctas);
    first_piece = true;
  }
  if (k.s >= k.end) return false;
  const int u = (int)((uint32_t)k.s / (uint32_t)n_it);
  w = kv_unit(a.g, first, whole + u, n_it);
  w.i0 = k.s - u * n_it;
  const int stop = w.i0 + (k.end - k.s);
  w.i1 = stop < n_it ? stop : n_it;
  w.slot = w.i1 - w.i0 == n_it ? -1 : first_piece ? 0 : 1;
  k.s += w.i1 - w.i0;
  return true;
}

template <int HD>
struct Dkv {
  static constexpr int kQ = 64;                     // query rows of a step
  static constexpr int kBlocks = HD / 64;
  static constexpr int kTile = kBlocks * kBlk128;   // K, V
  static constexpr int kQd = kBlocks * kBlk64;      // Q, dO
  static constexpr int kKvBufs = HD == 64 ? 2 : 1;
  static constexpr int kStages = HD == 64 ? 6 : 4;
  static constexpr int kStage = 2 * kQd;
  static constexpr int kKv = 0;                     // [buffer][K, V]
  static constexpr int kRing = kKvBufs * 2 * kTile;
  static constexpr int kStats = kRing + kStages * kStage;   // [stage][nlse, delta]
  static constexpr int kBar = kStats + kStages * 2 * kQ * 4;
  static constexpr int kBars = 2 * kKvBufs + 2 * kStages + 8 + 3;
  static constexpr int kSmem = kBar + kBars * 8 + 8 + 4 * kOrder + 1024;
  static_assert(kSmem <= 232448, "shared memory");
};

template <int HD, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
cross_dkdv_tc(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmG,
              const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
              const __grid_constant__ TcArgs a) {
  using F = Dkv<HD>;
  extern __shared__ uint8_t smem_raw[];
  if (!a.early) wait_for_launch_before();
  uint8_t* sp;
  const uint32_t base = align1024(smem_raw, &sp);
  auto sK = [&](int kb) { return base + F::kKv + 2 * kb * F::kTile; };
  auto sV = [&](int kb) { return base + F::kKv + (2 * kb + 1) * F::kTile; };
  auto sQ = [&](int st) { return base + F::kRing + st * F::kStage; };
  auto sG = [&](int st) { return base + F::kRing + st * F::kStage + F::kQd; };
  const uint32_t bars = base + F::kBar;
  auto kv_full = [&](int i) { return bars + 8u * i; };
  auto kv_empty = [&](int i) { return bars + 8u * (F::kKvBufs + i); };
  const uint32_t qbars = bars + 16u * F::kKvBufs;
  auto q_full = [&](int i) { return qbars + 8u * i; };
  auto q_empty = [&](int i) { return qbars + 8u * (F::kStages + i); };
  const uint32_t sbars = qbars + 16u * F::kStages;
  auto s_full = [&](int t) { return sbars + 8u * t; };
  auto p_full = [&](int t) { return sbars + 8u * (2 + t); };
  auto dp_full = [&](int t) { return sbars + 8u * (4 + t); };
  auto ds_full = [&](int t) { return sbars + 8u * (6 + t); };
  const uint32_t acc_full = sbars + 64u, acc_empty = sbars + 72u, done_bar = sbars + 80u;
  const uint32_t tslot = bars + 8u * F::kBars;
  uint32_t* tslot_ptr = reinterpret_cast<uint32_t*>(sp + F::kBar + 8 * F::kBars);
  // first[i]: key tiles of the sequences before i
  int* first = reinterpret_cast<int*>(sp + F::kBar + 8 * F::kBars + 8);

  const CrossGeom& g = a.g;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctas = (int)gridDim.x, cta = (int)blockIdx.x;
  const int64_t all_tiles = (g.kv_len + kRows - 1) / kRows;
  const bool table = kv_table(g);
  const int q_steps = a.q_pad / F::kQ;
  const int n_it = g.group * q_steps;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&tmQ);
    prefetch_tensormap(&tmG);
    prefetch_tensormap(&tmK);
    prefetch_tensormap(&tmV);
    for (int i = 0; i < F::kBars; ++i) {
      const uint32_t b = bars + 8u * i;
      const bool by_warps = b == p_full(0) || b == p_full(1) || b == ds_full(0) || b == ds_full(1);
      mbar_init(b, by_warps ? 4 : b == acc_empty ? 8 : 1);
    }
    fence_barrier_init();
  }
  if (warp == kMmaWarp) tmem_alloc(tslot, 512);
  if (table && warp == 0) tile_table(g, first);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tslot_ptr);
  auto tS = [&](int t) { return tmem + 128u * t; };
  auto tDp = [&](int t) { return tmem + 128u * t + 64u; };
  const uint32_t tDv = tmem + 256u, tDk = tmem + 256u + HD;
  const int units = kv_units(g, first);

  if (warp == kTmaWarp) {
    if (elect_one()) {
      bool ok = true;
      int gq = 0, ru = 0;
      KvWalk walk;
      KvUnit w;
      while (ok && kv_next(a, first, units, n_it, walk, w)) {
        if (w.i0 == w.i1) continue;
        if (w.len <= Dq<HD>::kKeys) wait_for_launch_before();  // dQ forms the delta of these
        const int kb = ru % F::kKvBufs;
        if (!mbar_wait(kv_empty(kb), (uint32_t)(((ru / F::kKvBufs) & 1) ^ 1), g.err)) break;
        mbar_expect_tx(kv_full(kb), 2 * F::kTile);
        for (int c = 0; c < F::kBlocks; ++c) {
          tma_load_4d(sK(kb) + c * kBlk128, &tmK, c * 64, w.kt * kRows, w.kvh * a.kh,
                      (int)w.b * a.kb, kv_full(kb));
          tma_load_4d(sV(kb) + c * kBlk128, &tmV, c * 64, w.kt * kRows, w.kvh * a.vh,
                      (int)w.b * a.vb, kv_full(kb));
        }
        for (int i = w.i0; i < w.i1; ++i, ++gq) {
          const int st = gq % F::kStages;
          if (!mbar_wait(q_empty(st), (uint32_t)(((gq / F::kStages) & 1) ^ 1), g.err)) {
            ok = false;
            break;
          }
          const int h = w.kvh * g.group + i / q_steps, q0 = i % q_steps * F::kQ;
          const int64_t at = (w.b * g.heads + h) * a.q_pad + q0;
          mbar_expect_tx(q_full(st), F::kStage + 2 * F::kQ * 4);
          for (int c = 0; c < F::kBlocks; ++c) {
            tma_load_4d(sQ(st) + c * kBlk64, &tmQ, c * 64, q0, h * a.qh, (int)w.b * a.qb, q_full(st));
            tma_load_4d(sG(st) + c * kBlk64, &tmG, c * 64, q0, h * a.dh, (int)w.b * a.db, q_full(st));
          }
          const uint32_t stats = base + F::kStats + st * 2 * F::kQ * 4;
          bulk_load(stats, a.nlse + at, F::kQ * 4, q_full(st));
          bulk_load(stats + F::kQ * 4, a.delta + at, F::kQ * 4, q_full(st));
        }
        ++ru;
      }
      for (int i = gq; i < gq + F::kStages && ok; ++i)
        ok = mbar_wait(q_empty(i % F::kStages), (uint32_t)(((i / F::kStages) & 1) ^ 1), g.err);
    }
  } else if (warp == kMmaWarp) {
    if (elect_one()) {
      constexpr uint32_t idS = idesc_bf16_f32(kRows, F::kQ, 0, 0);
      constexpr uint32_t idG = idesc_bf16_f32(kRows, HD, 0, 1);
      const uint64_t dk0 = desc_k(sK(0)), dv0 = desc_k(sV(0)), dq0 = desc_k(sQ(0)),
                     dg0 = desc_k(sG(0)), dqm0 = desc_mn(sQ(0), kBlk64),
                     dgm0 = desc_mn(sG(0), kBlk64);
      bool ok = true;
      int ru = 0;
      // the next step whose S^T / dP^T, and whose dV / dK, are issued: its ring
      // stage, its score buffer (alternating), and the parity of that buffer
      int sst = 0, gst = 0, dst = 0;
      uint32_t sph = 0, tb = 0, gp = 0, db = 0;
      auto q_wait = [&]() {
        if (!mbar_wait(q_full(sst), sph, g.err)) return false;
        tc_fence_after();
        return true;
      };
      auto issue_s = [&](uint32_t t, int kb) {
        const uint32_t ak = (uint32_t)kb * 2 * F::kTile;
        const uint64_t dk = desc_add(dk0, ak), dq = desc_add(dq0, (uint32_t)sst * F::kStage);
        const uint32_t d = tmem + 128u * t;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          mma_bf16_ss(d, desc_add(dk, k_step(kk, kBlk128)), desc_add(dq, k_step(kk, kBlk64)), idS,
                      kk > 0 ? 1u : 0u);
        mma_commit(s_full(t));
      };
      auto issue_dp = [&](uint32_t t, int kb) {
        const uint32_t ak = (uint32_t)kb * 2 * F::kTile;
        const uint64_t dv = desc_add(dv0, ak), dg = desc_add(dg0, (uint32_t)dst * F::kStage);
        const uint32_t d = tmem + 128u * t + 64u;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          mma_bf16_ss(d, desc_add(dv, k_step(kk, kBlk128)), desc_add(dg, k_step(kk, kBlk64)), idS,
                      kk > 0 ? 1u : 0u);
        mma_commit(dp_full(t));
        if (++dst == F::kStages) dst = 0;
      };
      auto s_next = [&]() {
        if (++sst == F::kStages) sst = 0, sph ^= 1u;
      };
      KvWalk walk;
      KvUnit next;
      bool have = kv_next(a, first, units, n_it, walk, next);
      while (ok && have) {
        const KvUnit w = next;
        if (w.i0 == w.i1) {
          have = kv_next(a, first, units, n_it, walk, next);
          continue;
        }
        const int kb = ru % F::kKvBufs;
        ok = mbar_wait(kv_full(kb), (uint32_t)((ru / F::kKvBufs) & 1), g.err);
        const int n = w.i1 - w.i0;
        for (int i = 0; i < 2 && i < n && ok; ++i) {
          ok = q_wait();
          if (!ok) break;
          issue_s(tb, kb);
          issue_dp(tb, kb);
          s_next();
          tb ^= 1u;
        }
        if (!ok) break;
        have = kv_next(a, first, units, n_it, walk, next);  // while the first products run
        for (int i = 0; i < n; ++i) {
          const uint32_t t = db;
          const uint32_t more = i > 0 ? 1u : 0u;
          const bool follows = i + 2 < n;
          const uint32_t aq = (uint32_t)gst * F::kStage, sc = tmem + 128u * t;
          ok = mbar_wait(p_full(t), gp, g.err) &&
               // the previous unit's dV and dK have been read
               (i > 0 || ru == 0 || mbar_wait(acc_empty, (uint32_t)((ru - 1) & 1), g.err)) &&
               (!follows || q_wait());
          if (!ok) break;
          tc_fence_after();
          {
            const uint64_t dgm = desc_add(dgm0, aq);
#pragma unroll
            for (int kk = 0; kk < F::kQ / 16; ++kk)
              mma_bf16_ts(tDv, sc + kk * 8, desc_add(dgm, kk * 2048), idG, kk > 0 ? 1u : more);
            if constexpr (SPLIT) {
#pragma unroll
              for (int kk = 0; kk < F::kQ / 16; ++kk)
                mma_bf16_ts(tDv, sc + 32u + kk * 8, desc_add(dgm, kk * 2048), idG, 1u);
            }
          }
          if (follows) issue_s(t, kb);  // behind dV, which reads P^T in the same columns
          ok = mbar_wait(ds_full(t), gp, g.err);
          if (!ok) break;
          tc_fence_after();
          {
            const uint64_t dqm = desc_add(dqm0, aq);
#pragma unroll
            for (int kk = 0; kk < F::kQ / 16; ++kk)
              mma_bf16_ts(tDk, sc + 64u + kk * 8, desc_add(dqm, kk * 2048), idG, kk > 0 ? 1u : more);
            if constexpr (SPLIT) {
#pragma unroll
              for (int kk = 0; kk < F::kQ / 16; ++kk)
                mma_bf16_ts(tDk, sc + 96u + kk * 8, desc_add(dqm, kk * 2048), idG, 1u);
            }
          }
          mma_commit(q_empty(gst));
          if (follows) {
            issue_dp(t, kb);
            s_next();
            tb ^= 1u;
          }
          if (++gst == F::kStages) gst = 0;
          gp ^= db;  // the parity of both buffers turns after the second one
          db ^= 1u;
        }
        if (!ok) break;
        ++ru;
        mma_commit(kv_empty(kb));
        mma_commit(acc_full);
      }
      mma_commit(done_bar);
      mbar_wait(done_bar, 0, g.err);
    }
  } else {
    const int t = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const float sl2 = scale_log2(g.scale);
    const unsigned long long sl22 = f2_pack(sl2, sl2);
    bool ok = true;
    int gs = 0, ru = 0;
    KvWalk walk;
    KvUnit next;
    bool have = kv_next(a, first, units, n_it, walk, next);
    while (have) {
      const KvUnit w = next;
      const int n_steps = w.i1 - w.i0;
      for (int i = 0; i < n_steps; ++i) {
        const int s = gs + i;
        if ((s & 1) != t) continue;
        const int st = s % F::kStages;
        if (ok && !mbar_wait(s_full(t), (uint32_t)((s >> 1) & 1), g.err)) ok = false;
        // the step's row terms came with its tiles
        if (ok && !mbar_wait(q_full(st), (uint32_t)((s / F::kStages) & 1), g.err)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) continue;
        tc_fence_after();
        const ulonglong2* nl =
            reinterpret_cast<const ulonglong2*>(sp + F::kStats + st * 2 * F::kQ * 4);
        const ulonglong2* dl = nl + F::kQ / 4;
        uint32_t vs[2][32];
        tmem_ld32(tS(t) + lanes, vs[0]);
        tmem_ld32(tS(t) + lanes + 32, vs[1]);
        tmem_wait_ld();
        auto terms = [&](const ulonglong2* p, int c) {
          return [p, c, x = ulonglong2{}](int e) mutable {
            if ((e & 1) == 0) x = p[c * 8 + (e >> 1)];
            return (e & 1) ? x.y : x.x;
          };
        };
        // P^T while dP^T is being computed
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          probs32(vs[c], sl22, terms(nl, c));
          uint32_t pp[16];
#pragma unroll
          for (int e = 0; e < 16; ++e)
            pp[e] = pack_bf16(__uint_as_float(vs[c][2 * e]), __uint_as_float(vs[c][2 * e + 1]));
          tmem_st16(tS(t) + lanes + 16 * c, pp);  // S^T is in registers
          if constexpr (SPLIT) {
            uint32_t pl[16];
            rest16(vs[c], pp, pl);
            tmem_st16(tS(t) + lanes + 32 + 16 * c, pl);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full(t));
        if (!mbar_wait(dp_full(t), (uint32_t)((s >> 1) & 1), g.err)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) continue;
        tc_fence_after();
        uint32_t vd[2][32];
        tmem_ld32(tDp(t) + lanes, vd[0]);
        tmem_ld32(tDp(t) + lanes + 32, vd[1]);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pd[16];
          if constexpr (SPLIT) {
            uint32_t pl[16];
            grads32_f32(vs[c], vd[c], terms(dl, c));
            pack32(vd[c], pd);
            rest16(vd[c], pd, pl);
            tmem_st16(tDp(t) + lanes + 32 + 16 * c, pl);
          } else {
            grads32(vs[c], vd[c], terms(dl, c), pd);
          }
          tmem_st16(tDp(t) + lanes + 16 * c, pd);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_full(t));
      }
      gs += n_steps;
      have = kv_next(a, first, units, n_it, walk, next);  // while the last products run
      // warpgroup 0 stores dV, warpgroup 1 dK
      const int64_t kj = (int64_t)w.kt * kRows + row;
      const bool in = kj < g.kv_len;
      __nv_bfloat16* dst =
          t == 0 ? static_cast<__nv_bfloat16*>(a.dv) + w.b * g.dvs[0] + w.kvh * g.dvs[1] + kj * g.dvs[2]
                 : static_cast<__nv_bfloat16*>(a.dk) + w.b * g.dks[0] + w.kvh * g.dks[1] + kj * g.dks[2];
      if (n_steps == 0) {
        if (in) zero_cols(dst, g.hd);
        continue;
      }
      if (ok && !mbar_wait(acc_full, (uint32_t)(ru & 1), g.err)) ok = false;
      ++ru;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) continue;
      tc_fence_after();
      const float mul = t == 0 ? 1.f : g.scale;
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t v[32];
        tmem_ld32((t == 0 ? tDv : tDk) + lanes + c * 32, v);
        tmem_wait_ld();
        if (c + 1 == HD / 32) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(acc_empty);
        }
        if (w.slot >= 0)
          store_piece32<HD>(piece_rows<HD>(a, cta, w.slot, t) + (int64_t)row * HD + c * 32, v);
        else if (kj < w.len && c * 32 < g.hd)
          store_cols32(dst + c * 32, v, mul, g.hd - c * 32);
      }
      if (in && kj >= w.len && w.slot < 0) zero_cols(dst, g.hd);
    }
    if (table) {  // the tiles without keys, which are no units
      for (int64_t i = cta; i < all_tiles * g.kv_heads * g.batch; i += ctas) {
        const int64_t kt = i % all_tiles, kvh = i / all_tiles % g.kv_heads,
                      b = i / all_tiles / g.kv_heads;
        if (kt < first[b + 1] - first[b]) continue;
        const int64_t kj = kt * kRows + row;
        if (kj >= g.kv_len) continue;
        zero_cols(t == 0 ? static_cast<__nv_bfloat16*>(a.dv) + b * g.dvs[0] + kvh * g.dvs[1] + kj * g.dvs[2]
                         : static_cast<__nv_bfloat16*>(a.dk) + b * g.dks[0] + kvh * g.dks[1] + kj * g.dks[2],
                  g.hd);
      }
    }
  }
  // This launch's end stands for that of the one before it too.
  wait_for_launch_before();
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// dV and dK of the units that a border of the steps cuts: a CTA per border and
// eighth of the 2 x 128 rows.
template <int HD>
__global__ void __launch_bounds__(256)
cross_dkdv_join(const __grid_constant__ TcArgs a, int ctas) {
  __shared__ int first[kOrder];
  __shared__ int list[kMostPieces], count;
  wait_for_launch_before();
  const CrossGeom& g = a.g;
  if (kv_table(g) && threadIdx.x < 32) tile_table(g, first);
  __syncthreads();
  const int n_it = g.group * (a.q_pad / Dkv<HD>::kQ);
  const int units = kv_units(g, first), whole = kv_whole(a, units, ctas);
  const int64_t total = (int64_t)(units - whole) * n_it, c = (int64_t)blockIdx.x + 1;
  const int64_t s = border(total, c, ctas);
  if (s >= total) return;
  const int64_t begin = s / n_it * n_it;
  // the unit begins here, or an earlier border has it
  if (begin == s || border(total, c - 1, ctas) > begin) return;
  const KvUnit w = kv_unit(g, first, whole + (int)(s / n_it), n_it);
  if (threadIdx.x == 0) count = list_pieces(total, ctas, c, begin, n_it, list);
  __syncthreads();
  constexpr int kVec = HD / 4;
  const int t = (int)blockIdx.y / 4;  // four CTAs a tile
  __nv_bfloat16* dst = t == 0 ? static_cast<__nv_bfloat16*>(a.dv) + w.b * g.dvs[0] + w.kvh * g.dvs[1]
                              : static_cast<__nv_bfloat16*>(a.dk) + w.b * g.dks[0] + w.kvh * g.dks[1];
  const int64_t step = t == 0 ? g.dvs[2] : g.dks[2];
#pragma unroll 2
  for (int i = threadIdx.x; i < 32 * kVec; i += 256) {
    const int row = (int)(blockIdx.y % 4) * 32 + i / kVec, col = i % kVec * 4;
    const int64_t kj = (int64_t)w.kt * kRows + row;
    if (col >= g.hd || kj >= g.kv_len) continue;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (kj < w.len) v = sum_pieces<HD>(a, list, count, t, row, col);
    store_grad4(dst + kj * step + col, v, t == 0 ? 1.f : g.scale);
  }
}

// ------------------------------------------------------------------ host side
// Map of a [batch, heads, positions, hd] view: boxes of 64 columns and `rows`
// positions. A batch or head stride of 0 becomes an extent of 1, and *bm or *hm
// 0: the kernels multiply the coordinate by it.
magma_status_t view_map(CUtensorMap* map, const void* p, int64_t hd, int64_t n, int64_t heads,
                        int64_t batch, const int64_t (&st)[3], int rows, int* bm, int* hm) {
  *bm = st[0] != 0;
  *hm = st[1] != 0;
  const uint64_t dims[4] = {(uint64_t)hd, (uint64_t)n, (uint64_t)(*hm ? heads : 1),
                            (uint64_t)(*bm ? batch : 1)};
  auto bytes = [](int64_t s) { return (uint64_t)(s ? 2 * s : 256); };
  const uint64_t strides[3] = {bytes(st[2]), bytes(st[1]), bytes(st[0])};
  const uint32_t box[4] = {64, (uint32_t)rows, 1, 1};
  return encode_tensor_map_nd(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p, 4, dims, strides, box,
                              CU_TENSOR_MAP_SWIZZLE_128B);
}

// Strides in 16-byte steps; positions may not share an address.
bool tc_strides(const void* p, const int64_t (&st)[3], int64_t n) {
  return aligned16(p) && st[0] % 8 == 0 && st[1] % 8 == 0 && st[2] % 8 == 0 &&
         (st[2] != 0 || n <= 1) && st[0] < (1LL << 38) && st[1] < (1LL << 38) &&
         st[2] < (1LL << 38);
}

TcArgs args_of(const CrossGeom& g) {
  TcArgs a{};
  a.g = g;
  a.n_qt = (int)ceil_div(g.q_len, kRows);
  a.n_pairs = (int)ceil_div((int64_t)g.group * a.n_qt, 2);
  a.n_split = 1;
  a.q_pad = (int)(ceil_div(g.q_len, 64) * 64);
  return a;
}

// Units and steps are counted in 32 bits.
bool fits32(int64_t a, int64_t b, int64_t c) { return (double)a * b * c < 1e9; }

template <int HD>
magma_status_t fwd_tc(const void* q, const void* k, const void* v, TcArgs a, cudaStream_t s) {
  const CrossGeom& g = a.g;
  CUtensorMap mq, mk, mv;
  if (magma_status_t st = view_map(&mq, q, g.hd, g.q_len, g.heads, g.batch, g.qs, kRows, &a.qb, &a.qh)) return st;
  if (magma_status_t st = view_map(&mk, k, g.hd, g.kv_len, g.kv_heads, g.batch, g.ks, kRows, &a.kb, &a.kh)) return st;
  if (magma_status_t st = view_map(&mv, v, g.hd, g.kv_len, g.kv_heads, g.batch, g.vs, kRows, &a.vb, &a.vh)) return st;
  if (magma_status_t st = cross_smem<cross_fwd_tc<HD>>(Fwd<HD>::kSmem)) return st;
  const int64_t units = (int64_t)a.n_pairs * a.n_split * g.kv_heads * g.batch;
  const unsigned ctas = (unsigned)std::min<int64_t>(units, num_sms());
  cross_fwd_tc<HD><<<ctas, kThreads, Fwd<HD>::kSmem, s>>>(mq, mk, mv, a);
  return check_launch("cross_fwd_tc");
}

// Whether the steps are dealt out: where whole units leave the CTAs idle for more
// than this many steps on average (lengths that differ: at least half a unit's).
// The pieces cost two stores of 128 rows and a second launch, about as long as 20
// steps.
constexpr int64_t kIdleSteps = 24;
bool deal(const CrossGeom& g, int64_t units, int64_t steps) {
  const int64_t n = num_sms();
  if (units > 16 * n || n > kMostPieces || steps > (1 << 18)) return false;
  const int64_t idle = steps * (ceil_div(units, n) * n - units) / n;
  return std::max(idle, g.lens != nullptr ? steps / 2 : 0) > kIdleSteps;
}
bool deal_dkdv(const CrossGeom& g) {
  return (g.lens == nullptr || g.batch < kOrder) &&
         deal(g, ceil_div(g.kv_len, kRows) * g.kv_heads * g.batch,
              (int64_t)g.group * ceil_div(g.q_len, 64));
}
bool deal_dq(const CrossGeom& g) {
  const TcArgs a = args_of(g);
  return (g.lens == nullptr || g.batch < kDealt) &&
         deal(g, (int64_t)a.n_pairs * g.kv_heads * g.batch, ceil_div(g.kv_len, 64));
}

// Whether P and dS go into the products as two BF16 terms, the rounded value and what
// it left: where no CTA has more than a step of dQ, and where dQ or dK has few rows.
// The sums of a large gradient have the error of their own rounding times sqrt(2)
// with single terms; that of a small one scatters around it (measured: up to 1.6; 256
// rows of 32 under 16 sources of 65 keys 1.53), and in small calls the second
// product hides in the launches' latency (2 x 8 heads, 128 x 128: 15.2 and 16.2 us at head
// size 64, 17.9 and 19.5 at 128). With more steps it costs a seventh to a fifth
// (2 x 16 heads, 512 x 512: 27.4 and 31.7 us; 8 x 16 heads, 512 x 1024: 105 and 125).
bool two_terms(const CrossGeom& g) {
  const TcArgs a = args_of(g);
  return g.batch * g.heads * g.q_len <= 1024 || g.batch * g.kv_heads * g.kv_len <= 1024 ||
         (double)a.n_pairs * g.kv_heads * g.batch * ceil_div(g.kv_len, 64) <= (double)num_sms();
}

template <int HD, bool SPLIT>
magma_status_t bwd_tc(const void* q, const void* k, const void* v, const void* d_o, float* piece,
                      TcArgs a, cudaStream_t s) {
  const CrossGeom& g = a.g;
  CUtensorMap mq, mg, mk, mv;
  {  // dQ first: it writes the delta of short sources, which dK reads
    using F = Dq<HD>;
    if (magma_status_t st = view_map(&mq, q, g.hd, g.q_len, g.heads, g.batch, g.qs, kRows, &a.qb, &a.qh)) return st;
    if (magma_status_t st = view_map(&mg, d_o, g.hd, g.q_len, g.heads, g.batch, g.dos, kRows, &a.db, &a.dh)) return st;
    if (magma_status_t st = view_map(&mk, k, g.hd, g.kv_len, g.kv_heads, g.batch, g.ks, F::kKeys, &a.kb, &a.kh)) return st;
    if (magma_status_t st = view_map(&mv, v, g.hd, g.kv_len, g.kv_heads, g.batch, g.vs, F::kKeys, &a.vb, &a.vh)) return st;
    if (magma_status_t st = cross_smem<cross_dq_tc<HD, SPLIT>>(F::kSmem)) return st;
    const int64_t units = (int64_t)a.n_pairs * g.kv_heads * g.batch;
    a.piece = deal_dq(g) ? piece : nullptr;
    const unsigned ctas = (unsigned)(a.piece ? num_sms() : std::min<int64_t>(units, num_sms()));
    if (magma_status_t st = launch_after(cross_dq_tc<HD, SPLIT>, dim3(ctas), kThreads, F::kSmem, s,
                                         "cross_dq_tc", mq, mg, mk, mv, a))
      return st;
    if (a.piece)
      if (magma_status_t st = launch_after(cross_dq_join<HD>, dim3(ctas - 1, 8), 256, 0, s,
                                           "cross_dq_join", a, (int)ctas))
        return st;
  }
  using F = Dkv<HD>;
  if (magma_status_t st = view_map(&mq, q, g.hd, g.q_len, g.heads, g.batch, g.qs, F::kQ, &a.qb, &a.qh)) return st;
  if (magma_status_t st = view_map(&mg, d_o, g.hd, g.q_len, g.heads, g.batch, g.dos, F::kQ, &a.db, &a.dh)) return st;
  if (magma_status_t st = view_map(&mk, k, g.hd, g.kv_len, g.kv_heads, g.batch, g.ks, kRows, &a.kb, &a.kh)) return st;
  if (magma_status_t st = view_map(&mv, v, g.hd, g.kv_len, g.kv_heads, g.batch, g.vs, kRows, &a.vb, &a.vh)) return st;
  if (magma_status_t st = cross_smem<cross_dkdv_tc<HD, SPLIT>>(F::kSmem)) return st;
  a.early = a.piece == nullptr;
  const int64_t units = ceil_div(g.kv_len, kRows) * g.kv_heads * g.batch;
  a.piece = deal_dkdv(g) ? piece : nullptr;
  const unsigned ctas = (unsigned)(a.piece ? num_sms() : std::min<int64_t>(units, num_sms()));
  if (magma_status_t st = launch_after(cross_dkdv_tc<HD, SPLIT>, dim3(ctas), kThreads, F::kSmem, s,
                                       "cross_dkdv_tc", mq, mg, mk, mv, a))
    return st;
  if (a.piece == nullptr) return MAGMA_OK;
  return launch_after(cross_dkdv_join<HD>, dim3(ctas - 1, 8), 256, 0, s, "cross_dkdv_join", a,
                      (int)ctas);
}

}  // namespace

// Without sequences or query heads there is no grid to launch; the FMA-pipe kernels
// write what such a call has to write (zeros to dK and dV).
bool cross_tc_fwd_supported(const void* q, const void* k, const void* v, const void* o,
                            const CrossGeom& g, magma_dtype_t dtype) {
  return dtype == MAGMA_DTYPE_BF16 && g.hd % 8 == 0 && g.kv_len > 0 && g.q_len > 0 &&
         g.batch > 0 && g.heads > 0 &&
         tc_strides(q, g.qs, g.q_len) && tc_strides(k, g.ks, g.kv_len) &&
         tc_strides(v, g.vs, g.kv_len) && tc_strides(o, g.os, g.q_len) &&
         fits32(g.batch, g.kv_heads, ceil_div(g.kv_len, kRows)) &&
         fits32(g.batch, g.heads, ceil_div(g.q_len, 64));
}

bool cross_tc_bwd_supported(const void* q, const void* k, const void* v, const void* o,
                            const void* d_o, const void* dq, const void* dk, const void* dv,
                            const CrossGeom& g, magma_dtype_t dtype) {
  return cross_tc_fwd_supported(q, k, v, o, g, dtype) && tc_strides(d_o, g.dos, g.q_len) &&
         tc_strides(dq, g.dqs, g.q_len) && tc_strides(dk, g.dks, g.kv_len) &&
         tc_strides(dv, g.dvs, g.kv_len);
}

// Parts of a source: as many as fill the SMs, at least two key tiles each (a
// part costs its share of the join: one F32 row per query and part). Unsplit, and in
// parts of at least two tiles, one, four: 2 heads of 64, 100 x 6000, 57, 13, 12 and 14
// us; 8 heads of 128, 256 x 4096, 58, 24, 25 and 21; 16 heads of 64, 128 x 1024, 14, 11, 11
// and 13. Short sources lose by it: 4 x 8 heads of 128, 256 x 512, 14, 20, 21 and 14.
static int64_t wanted_splits(const CrossGeom& g) {
  const TcArgs a = args_of(g);
  const int64_t units = (int64_t)a.n_pairs * g.kv_heads * g.batch;
  const int64_t tiles = ceil_div(g.kv_len, kRows);
  return std::max<int64_t>(1, std::min<int64_t>(num_sms() / std::max<int64_t>(units, 1), tiles / 2));
}

size_t cross_tc_fwd_workspace(const CrossGeom& g) {
  const int64_t n = wanted_splits(g);
  return n <= 1 ? 0 : (size_t)n * g.batch * g.heads * g.q_len * (g.hd + 1) * sizeof(float);
}

magma_status_t cross_fwd_tc_run(const void* q, const void* k, const void* v, void* o, float* lse,
                                const CrossGeom& g, void* workspace, size_t workspace_bytes,
                                cudaStream_t s) {
  TcArgs a = args_of(g);
  a.o = o;
  a.lse = lse;
  const int64_t rows = g.batch * g.heads * g.q_len;
  const size_t each = (size_t)rows * (g.hd + 1) * sizeof(float);
  if (workspace != nullptr && aligned16(workspace))
    a.n_split = (int)std::max<int64_t>(1, std::min<int64_t>(wanted_splits(g), workspace_bytes / each));
  if (a.n_split > 1) {
    a.part = static_cast<float*>(workspace);
    a.part_lse = a.part + (size_t)a.n_split * rows * g.hd;
  }
  if (magma_status_t st = g.hd <= 64 ? fwd_tc<64>(q, k, v, a, s) : fwd_tc<128>(q, k, v, a, s))
    return st;
  if (a.n_split == 1) return MAGMA_OK;
  return cross_join_parts(a.part, a.part_lse, o, lse, g, a.n_split, MAGMA_DTYPE_BF16, s);
}

// The row terms, then the pieces: two slots of two tiles a CTA. (Room for them is
// asked for with and without lengths, which the query does not know of.)
static size_t row_bytes(const CrossGeom& g) {
  return 2 * sizeof(float) * (size_t)g.batch * g.heads * (ceil_div(g.q_len, 64) * 64);
}
size_t cross_tc_bwd_workspace(const CrossGeom& g) {
  static const int32_t some = 0;
  CrossGeom l = g;
  l.lens = &some;
  const bool pieces = deal_dkdv(g) || deal_dq(g) || deal_dkdv(l) || deal_dq(l);
  return row_bytes(g) +
         (pieces ? (size_t)num_sms() * 4 * kRows * (g.hd <= 64 ? 64 : 128) * sizeof(float) : 0);
}

magma_status_t cross_bwd_tc_run(const void* q, const void* k, const void* v, const void* o,
                                const void* d_o, const float* lse, void* dq, void* dk, void* dv,
                                void* workspace, const CrossGeom& g, cudaStream_t s) {
  TcArgs a = args_of(g);
  const int64_t rows = g.batch * g.heads * a.q_pad;
  float* nlse = static_cast<float*>(workspace);
  float* delta = nlse + rows;
  a.nlse = nlse;
  a.delta = delta;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  cross_rows<<<(unsigned)(rows / 64), 128, 0, s>>>(
      static_cast<const __nv_bfloat16*>(o), static_cast<const __nv_bfloat16*>(d_o), lse, nlse, delta,
      g, a.q_pad);
  if (magma_status_t st = check_launch("cross_rows")) return st;
  float* piece = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + row_bytes(g));
  auto* run = two_terms(g) ? (g.hd <= 64 ? bwd_tc<64, true> : bwd_tc<128, true>)
                           : (g.hd <= 64 ? bwd_tc<64, false> : bwd_tc<128, false>);
  return run(q, k, v, d_o, piece, a, s);
}

}  // namespace magma
