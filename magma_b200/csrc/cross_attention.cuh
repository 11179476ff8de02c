// What the cross-attention kernels share: the geometry of a call and the
// hand-over between the entry points and the kernel files.
#pragma once

#include "common.cuh"

namespace magma {

// Queries [B, H, Sq, D] over keys and values [B, Hkv, Skv, D]; query head h
// reads key head h / group. Strides (batch, head, position) are in elements,
// the last dimension is contiguous. lens[b] keys of sequence b are there (all
// of them where lens is NULL).
struct CrossGeom {
  int64_t batch, heads, kv_heads, q_len, kv_len;
  int group, hd;
  float scale;
  const int32_t* lens;
  int64_t qs[3], ks[3], vs[3], os[3];
  // gradients: of dO, dQ, dK, dV
  int64_t dos[3], dqs[3], dks[3], dvs[3];
  int* err;
};

// Keys of sequence b; a length outside [0, kv_len] is clamped and reported.
__device__ __forceinline__ int64_t cross_len(const CrossGeom& g, int64_t b) {
  if (g.lens == nullptr) return g.kv_len;
  const int64_t n = g.lens[b];
  if (n < 0 || n > g.kv_len) {
    set_device_error(g.err, kDevErrBadIndex);
    return n < 0 ? 0 : g.kv_len;
  }
  return n;
}

// Lets a kernel use `bytes` of dynamic shared memory, asked once per kernel and
// device (`Kernel` is a type of its own for each kernel).
template <auto Kernel>
magma_status_t cross_smem(int bytes) {
  static bool done[64] = {};
  int dev = 0;
  if (magma_status_t st = cuda_status(cudaGetDevice(&dev), "cudaGetDevice")) return st;
  if (dev < 64 && done[dev]) return MAGMA_OK;
  if (magma_status_t st = cuda_status(
          cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
          "cross attention shared memory"))
    return st;
  if (dev < 64) done[dev] = true;
  return MAGMA_OK;
}

// cross_attention_simt.cu: any types, strides and head sizes up to 128. The
// forward pass takes less workspace or none.
size_t cross_simt_fwd_workspace(const CrossGeom& g);
magma_status_t cross_fwd_simt(const void* q, const void* k, const void* v, void* o, float* lse,
                              const CrossGeom& g, magma_dtype_t dtype, void* workspace,
                              size_t workspace_bytes, cudaStream_t s);
size_t cross_simt_bwd_workspace(const CrossGeom& g);
magma_status_t cross_bwd_simt(const void* q, const void* k, const void* v, const void* o,
                              const void* d_o, const float* lse, void* dq, void* dk, void* dv,
                              const CrossGeom& g, magma_dtype_t dtype, void* workspace,
                              size_t workspace_bytes, cudaStream_t s);

// cross_attention_step.cu: few query rows per key head (_rows: as far as sizes
// say), 16-byte aligned positions.
bool cross_step_rows(const CrossGeom& g, magma_dtype_t dtype);
bool cross_step_supported(const void* q, const void* k, const void* v, const void* o,
                          const CrossGeom& g, magma_dtype_t dtype);
size_t cross_step_workspace(const CrossGeom& g, magma_dtype_t dtype);
magma_status_t cross_step_run(const void* q, const void* k, const void* v, void* o, float* lse,
                              const CrossGeom& g, magma_dtype_t dtype, void* workspace,
                              size_t workspace_bytes, cudaStream_t s);

// cross_attention_join.cu: parts [n_part][batch][heads][q_len][hd] and their lse.
magma_status_t cross_join_parts(const float* part, const float* part_lse, void* o, float* lse,
                                const CrossGeom& g, int n_part, magma_dtype_t dtype,
                                cudaStream_t s);

// cross_attention_tc.cu: BF16, head sizes that are multiples of 8, 16-byte
// aligned positions. Workspaces in bytes; the forward pass takes less or none.
bool cross_tc_fwd_supported(const void* q, const void* k, const void* v, const void* o,
                            const CrossGeom& g, magma_dtype_t dtype);
size_t cross_tc_fwd_workspace(const CrossGeom& g);
magma_status_t cross_fwd_tc_run(const void* q, const void* k, const void* v, void* o, float* lse,
                                const CrossGeom& g, void* workspace, size_t workspace_bytes,
                                cudaStream_t s);
bool cross_tc_bwd_supported(const void* q, const void* k, const void* v, const void* o,
                            const void* d_o, const void* dq, const void* dk, const void* dv,
                            const CrossGeom& g, magma_dtype_t dtype);
size_t cross_tc_bwd_workspace(const CrossGeom& g);
magma_status_t cross_bwd_tc_run(const void* q, const void* k, const void* v, const void* o,
                                const void* d_o, const float* lse, void* dq, void* dk, void* dv,
                                void* workspace, const CrossGeom& g, cudaStream_t s);

}  // namespace magma
