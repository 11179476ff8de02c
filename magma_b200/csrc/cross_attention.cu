// C-ABI entry points of cross attention: argument checks and dispatch.
#include <algorithm>
#include <cmath>

#include "cross_attention.cuh"
#include "memory_views.cuh"

using namespace magma;

namespace {

// Strides of a [d0, d1, d2, hd] tensor. An output's positions may not share
// memory: taken from the smallest stride up, each must step over all that the
// smaller ones span.
magma_status_t set_strides(const char* fn, const char* what, const int64_t* from, int64_t (&to)[3],
                           bool output, int64_t d0, int64_t d1, int64_t d2, int64_t hd) {
  MAGMA_REQUIRE(from != nullptr, "%s: NULL strides of %s", fn, what);
  const int64_t dims[3] = {d0, d1, d2};
  for (int i = 0; i < 3; ++i) {
    MAGMA_REQUIRE(from[i] >= 0 && from[i] < (1LL << 40), "%s: stride %lld of %s", fn,
                  (long long)from[i], what);
    to[i] = dims[i] > 1 ? from[i] : 0;
  }
  if (!output || d0 == 0 || d1 == 0 || d2 == 0) return MAGMA_OK;
  int order[3] = {0, 1, 2};
  std::sort(order, order + 3, [&](int a, int b) { return to[a] < to[b]; });
  int64_t span = hd;
  for (int i : order) {
    if (dims[i] <= 1) continue;
    MAGMA_REQUIRE(to[i] >= span, "%s: positions of %s share memory (stride %lld over %lld)", fn,
                  what, (long long)to[i], (long long)span);
    span += to[i] * (dims[i] - 1);
  }
  return MAGMA_OK;
}

MemView view(const void* p, const CrossGeom& g, int64_t heads, int64_t len, const int64_t (&st)[3],
             magma_dtype_t dtype) {
  const int64_t e = (int64_t)dtype_size(dtype);
  return {p, g.hd * e, {g.batch, heads, len}, {st[0] * e, st[1] * e, st[2] * e}};
}
MemView lse_view(const float* lse, const CrossGeom& g) {
  return {lse, 4 * g.q_len, {g.batch, g.heads, 1}, {4 * g.heads * g.q_len, 4 * g.q_len, 0}};
}
MemView lens_view(const CrossGeom& g) { return {g.lens, 4 * g.batch}; }

CrossGeom sizes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t q_len, int64_t kv_len,
                int64_t hd) {
  CrossGeom g{};
  g.batch = batch;
  g.heads = heads;
  g.kv_heads = kv_heads;
  g.q_len = q_len;
  g.kv_len = kv_len;
  g.group = kv_heads ? (int)(heads / kv_heads) : 0;
  g.hd = (int)hd;
  return g;
}

// Lengths are padded to multiples of 64 in 32-bit counters.
constexpr int64_t kMaxLen = (1LL << 31) - 64;

// Whether a workspace query is about a call that launches anything.
bool has_work(int64_t batch, int64_t heads, int64_t kv_heads, int64_t q_len, int64_t kv_len,
              int64_t hd) {
  return batch > 0 && heads > 0 && kv_heads > 0 && q_len > 0 && kv_len > 0 && hd > 0 && hd <= 128 &&
         batch < 65536 && heads < 65536 && heads % kv_heads == 0 && q_len <= kMaxLen &&
         kv_len <= kMaxLen;
}

magma_status_t geometry(const char* fn, const int32_t* kv_lens, int64_t batch, int64_t heads,
                        int64_t kv_heads, int64_t q_len, int64_t kv_len, int64_t hd, float scale,
                        magma_dtype_t dtype, CrossGeom* g) {
  MAGMA_REQUIRE(batch >= 0 && heads >= 0 && kv_heads >= 0 && q_len >= 0 && kv_len >= 0,
                "%s: negative size", fn);
  MAGMA_REQUIRE(batch < 65536 && heads < 65536, "%s: batch and heads must be < 65536", fn);
  MAGMA_REQUIRE(q_len <= kMaxLen && kv_len <= kMaxLen, "%s: lengths must be at most 2^31 - 64", fn);
  MAGMA_REQUIRE(hd >= 1 && hd <= 128, "%s: head_dim %lld outside [1, 128]", fn, (long long)hd);
  MAGMA_REQUIRE(kv_heads == 0 ? heads == 0 : heads % kv_heads == 0,
                "%s: heads (%lld) must be a multiple of kv_heads (%lld)", fn, (long long)heads,
                (long long)kv_heads);
  MAGMA_REQUIRE(is_float_dtype(dtype), "%s: dtype must be F32 or BF16", fn);
  MAGMA_REQUIRE(std::isfinite(scale) && scale >= 0.f, "%s: scale must be finite and not negative",
                fn);
  *g = sizes(batch, heads, kv_heads, q_len, kv_len, hd);
  g->scale = scale;
  g->lens = kv_lens;
  g->err = device_error_word();
  return MAGMA_OK;
}

}  // namespace

extern "C" {

size_t magma_cross_attention_fwd_workspace_size(int64_t batch, int64_t heads, int64_t kv_heads,
                                                int64_t q_len, int64_t kv_len, int64_t head_dim,
                                                magma_dtype_t dtype) {
  if (!has_work(batch, heads, kv_heads, q_len, kv_len, head_dim)) return 0;
  CrossGeom g = sizes(batch, heads, kv_heads, q_len, kv_len, head_dim);
  if (cross_step_rows(g, dtype)) return cross_step_workspace(g, dtype);
  return dtype == MAGMA_DTYPE_BF16 && head_dim % 8 == 0 ? cross_tc_fwd_workspace(g)
                                                        : cross_simt_fwd_workspace(g);
}

magma_status_t magma_cross_attention_fwd(const void* q, const void* k, const void* v, void* o,
                                         float* lse, const int32_t* kv_lens, int64_t batch,
                                         int64_t heads, int64_t kv_heads, int64_t q_len,
                                         int64_t kv_len, int64_t head_dim,
                                         const int64_t* q_strides, const int64_t* k_strides,
                                         const int64_t* v_strides, const int64_t* o_strides,
                                         float scale, magma_dtype_t dtype, void* workspace,
                                         size_t workspace_bytes, void* stream) {
  const char* fn = "magma_cross_attention_fwd";
  CrossGeom g{};
  if (magma_status_t st = geometry(fn, kv_lens, batch, heads, kv_heads, q_len, kv_len, head_dim,
                                   scale, dtype, &g))
    return st;
  if (magma_status_t st = set_strides(fn, "q", q_strides, g.qs, false, batch, heads, q_len, head_dim)) return st;
  if (magma_status_t st = set_strides(fn, "k", k_strides, g.ks, false, batch, kv_heads, kv_len, head_dim)) return st;
  if (magma_status_t st = set_strides(fn, "v", v_strides, g.vs, false, batch, kv_heads, kv_len, head_dim)) return st;
  if (magma_status_t st = set_strides(fn, "o", o_strides, g.os, true, batch, heads, q_len, head_dim)) return st;
  if (batch == 0 || heads == 0 || q_len == 0) return MAGMA_OK;
  MAGMA_REQUIRE(q && o && (kv_len == 0 || (k && v)), "%s: NULL pointer", fn);
  const void* tensors[] = {q, k, v, o};
  for (const void* x : tensors)
    MAGMA_REQUIRE(on_element(x, dtype_size(dtype)), "%s: an address off its elements", fn);
  MAGMA_REQUIRE(on_element(lse, 4) && on_element(kv_lens, 4), "%s: an address off its elements", fn);
  const MemView inputs[] = {view(q, g, heads, q_len, g.qs, dtype),
                            view(k, g, kv_heads, kv_len, g.ks, dtype),
                            view(v, g, kv_heads, kv_len, g.vs, dtype), lens_view(g)};
  const MemView ov = view(o, g, heads, q_len, g.os, dtype), lv = lse_view(lse, g);
  for (const MemView& x : inputs) {
    MAGMA_REQUIRE(!share_memory(ov, x), "%s: o shares memory with an input", fn);
    MAGMA_REQUIRE(!share_memory(lv, x), "%s: lse shares memory with an input", fn);
  }
  MAGMA_REQUIRE(!share_memory(ov, lv), "%s: o and lse share memory", fn);
  if (cross_step_supported(q, k, v, o, g, dtype))
    return cross_step_run(q, k, v, o, lse, g, dtype, workspace, workspace_bytes,
                          (cudaStream_t)stream);
  if (cross_tc_fwd_supported(q, k, v, o, g, dtype))
    return cross_fwd_tc_run(q, k, v, o, lse, g, workspace, workspace_bytes, (cudaStream_t)stream);
  return cross_fwd_simt(q, k, v, o, lse, g, dtype, workspace, workspace_bytes,
                        (cudaStream_t)stream);
}

size_t magma_cross_attention_bwd_workspace_size(int64_t batch, int64_t heads, int64_t kv_heads,
                                                int64_t q_len, int64_t kv_len, int64_t head_dim,
                                                magma_dtype_t dtype) {
  if (batch <= 0 || heads <= 0 || q_len <= 0) return 0;
  // without keys dQ = 0 and nothing but delta is formed
  if (!has_work(batch, heads, kv_heads, q_len, kv_len, head_dim))
    return (sizeof(float) * (size_t)batch * (size_t)heads * (size_t)q_len + 15) / 16 * 16;
  const CrossGeom g = sizes(batch, heads, kv_heads, q_len, kv_len, head_dim);
  return dtype == MAGMA_DTYPE_BF16 && head_dim % 8 == 0 ? cross_tc_bwd_workspace(g)
                                                        : cross_simt_bwd_workspace(g);
}

magma_status_t magma_cross_attention_bwd(
    const void* q, const void* k, const void* v, const void* o, const void* d_o, const float* lse,
    const int32_t* kv_lens, void* dq, void* dk, void* dv, int64_t batch, int64_t heads,
    int64_t kv_heads, int64_t q_len, int64_t kv_len, int64_t head_dim, const int64_t* q_strides,
    const int64_t* k_strides, const int64_t* v_strides, const int64_t* o_strides,
    const int64_t* do_strides, const int64_t* dq_strides, const int64_t* dk_strides,
    const int64_t* dv_strides, float scale, magma_dtype_t dtype, void* workspace,
    size_t workspace_bytes, void* stream) {
  const char* fn = "magma_cross_attention_bwd";
  CrossGeom g{};
  if (magma_status_t st = geometry(fn, kv_lens, batch, heads, kv_heads, q_len, kv_len, head_dim,
                                   scale, dtype, &g))
    return st;
  struct {
    const char* what;
    const int64_t* from;
    int64_t (&to)[3];
    bool output, keys;
  } all[] = {{"q", q_strides, g.qs, false, false},    {"k", k_strides, g.ks, false, true},
             {"v", v_strides, g.vs, false, true},     {"o", o_strides, g.os, false, false},
             {"d_o", do_strides, g.dos, false, false}, {"dq", dq_strides, g.dqs, true, false},
             {"dk", dk_strides, g.dks, true, true},   {"dv", dv_strides, g.dvs, true, true}};
  for (auto& x : all)
    if (magma_status_t st = set_strides(fn, x.what, x.from, x.to, x.output, batch,
                                        x.keys ? kv_heads : heads, x.keys ? kv_len : q_len, head_dim))
      return st;
  const bool has_q = batch && heads && q_len, has_k = batch && kv_heads && kv_len;
  MAGMA_REQUIRE(!has_q || (q && o && d_o && lse && dq), "%s: NULL pointer", fn);
  MAGMA_REQUIRE(!has_k || (k && v && dk && dv), "%s: NULL pointer", fn);
  const void* tensors[] = {q, k, v, o, d_o, dq, dk, dv};
  for (const void* x : tensors)
    MAGMA_REQUIRE(on_element(x, dtype_size(dtype)), "%s: an address off its elements", fn);
  MAGMA_REQUIRE(on_element(lse, 4) && on_element(kv_lens, 4), "%s: an address off its elements", fn);
  const MemView inputs[] = {view(q, g, heads, q_len, g.qs, dtype),
                            view(k, g, kv_heads, kv_len, g.ks, dtype),
                            view(v, g, kv_heads, kv_len, g.vs, dtype),
                            view(o, g, heads, q_len, g.os, dtype),
                            view(d_o, g, heads, q_len, g.dos, dtype), lse_view(lse, g), lens_view(g)};
  const MemView grads[] = {view(dq, g, heads, q_len, g.dqs, dtype),
                           view(dk, g, kv_heads, kv_len, g.dks, dtype),
                           view(dv, g, kv_heads, kv_len, g.dvs, dtype)};
  for (int i = 0; i < 3; ++i) {
    for (const MemView& x : inputs)
      MAGMA_REQUIRE(!share_memory(grads[i], x), "%s: a gradient shares memory with an input", fn);
    for (int j = 0; j < i; ++j)
      MAGMA_REQUIRE(!share_memory(grads[i], grads[j]), "%s: two gradients share memory", fn);
  }
  const size_t need = magma_cross_attention_bwd_workspace_size(batch, heads, kv_heads, q_len,
                                                               kv_len, head_dim, dtype);
  MAGMA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)),
                "%s: a 16-byte aligned workspace of %zu bytes is needed", fn, need);
  if (cross_tc_bwd_supported(q, k, v, o, d_o, dq, dk, dv, g, dtype))
    return cross_bwd_tc_run(q, k, v, o, d_o, lse, dq, dk, dv, workspace, g, (cudaStream_t)stream);
  return cross_bwd_simt(q, k, v, o, d_o, lse, dq, dk, dv, g, dtype, workspace, workspace_bytes,
                        (cudaStream_t)stream);
}

}  // extern "C"
