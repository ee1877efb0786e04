// Host side shared by the cross-attention entry points: argument block of the C interface, tensor maps.
#pragma once
#include "cross_attention.cuh"
#include <math.h>

// Packed field by field in native_cross_attention.py; strides in elements.
struct SbCrossAttention {
  const void *q, *k, *v;
  long long q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  const int* lengths;
  const uint8_t* mask;
  int type;                            // 0 = bf16, 1 = fp16
  int M, G, rep, Tq, Tk, Hk, D;
  float scale;
};

// Checks the block and fills the kernels' arguments; 0, SB_BAD_ARGUMENT or a negative code.
int sb_xattn_args(const SbCrossAttention* g, XAttnArgs* a);
// [T, heads, batch] rows of D 16-bit elements as a 4-D map (D, T, heads, batch) with a {64, box, 1, 1} box, 128-byte swizzle, zeros outside.
int sb_rows_map(CUtensorMap* map, const void* ptr, int type, int D, int T, int heads, int batch, long long st, long long sh, long long sb, int box);
// A grid of one block per result tile, or of a cluster per tile whose blocks share the tile's summed axis.
struct SbClusterLaunch {
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute attr[1];
  SbClusterLaunch(long long tiles, int splits, int threads, int smem, cudaStream_t stream) {
    config.gridDim = dim3((unsigned)(tiles * splits));
    config.blockDim = dim3((unsigned)threads);
    config.dynamicSmemBytes = (size_t)smem;
    config.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = splits > 1 ? 1 : 0;
  }
};
// How to run `tiles` result tiles, each a sum over `steps` steps: the first `whole` by a block each, the rest by clusters of `splits` blocks.
// Clusters of 2, 4 or 8 take the tiles that do not fill the SMs (all of them, or those behind the last full wave) where that makes the
// schedule shorter.  `own`, `join`: what a block takes besides its steps, and with others for the join, in steps.  (Full waves stay
// whole: a split costs there.  dq, 4 x 1024 queries, 7500 keys, 256 tiles: 1 / 2 blocks a tile 157 / 194 us.)
struct SbTilePlan { long long whole; int splits; };
SbTilePlan sb_plan_tiles(const void* kernel, int threads, int smem, long long tiles, int steps, int own, int join);
template <typename... P, typename... Q>
int sb_run_tiles(const SbTilePlan& plan, long long tiles, int threads, int smem, cudaStream_t stream, void (*kernel)(P...), const Q&... args) {
  if (plan.whole > 0) {
    SbClusterLaunch l(plan.whole, 1, threads, smem, stream);
    const int rc = (int)cudaLaunchKernelEx(&l.config, kernel, args..., 0ll, 1);
    if (rc) return rc;
  }
  if (plan.whole == tiles) return 0;
  SbClusterLaunch l(tiles - plan.whole, plan.splits, threads, smem, stream);
  return (int)cudaLaunchKernelEx(&l.config, kernel, args..., plan.whole, plan.splits);
}
// Dynamic shared memory of a kernel, set once per kernel and device.
int sb_allow_smem(const void* kernel, int bytes);

// Whether a call has few enough query rows per key head for the decoding-step kernel (step_attention.cu).
bool sb_few_rows(const SbCrossAttention* g);
int sb_step_cross_attention(const SbCrossAttention* g, void* out, void* rest, float* lse, void* ws, cudaStream_t stream);
