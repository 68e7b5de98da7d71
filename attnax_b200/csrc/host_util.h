// Host helpers shared by the library's translation units.
#pragma once
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <cstddef>

#include "../../include/attnb200.h"

namespace attnb200 {

inline size_t dtype_size(attn_dtype_t t) { return t == ATTN_F32 ? 4 : 2; }
inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// cuTensorMapEncodeTiled of the running driver (null without one).
PFN_cuTensorMapEncodeTiled_v12000 encode_fn();

// Counts `n` kernel launches and reports the launch error state.
int launch_status(int n = 1);

// Launches `kernel` so that it may start while the previous kernel of the
// stream drains; it must call pdl_wait_previous() before it reads or writes
// anything that one touches.
template <typename... P, typename... A>
inline void launch_overlapped(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, P(args)...);  // (the error state is read by launch_status)
}

// Launches `kernel` in clusters of `cluster` CTAs along y.
template <typename... P, typename... A>
inline void launch_cluster_y(void (*kernel)(P...), int cluster, dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                             const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 1;
  at[0].val.clusterDim.y = cluster;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// 4-D tiled map over a (B, H, S, D) tensor (see attnb200.cu).
bool make_tmap(CUtensorMap* m, attn_dtype_t dt, const void* ptr, int B, int H, int S, int D, const int64_t* s,
               int box_rows);
// 3-D map over a page pool (see attnb200.cu).
bool make_pool_tmap(CUtensorMap* m, attn_dtype_t dt, const void* pool, long long tokens, int heads_kv, int head_dim,
                    int box_tokens);

// Each translation unit has its own device status words (sm100.cuh); these
// read and clear those of the others for attn_device_status.
bool rows_take_status(int* status, int* notice);
bool pages_take_status(int* status, int* notice);
bool rotary_take_status(int* status, int* notice);
bool attend8_take_status(int* status, int* notice);

}  // namespace attnb200
