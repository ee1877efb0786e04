// Host side shared by the cross-attention entry points: argument block of the C interface, tensor maps.
#pragma once
#include "cross_attention.cuh"
#include <math.h>

// Mirrored by a ctypes structure in native_cross_attention.py; strides in elements.
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
// Dynamic shared memory of a kernel, set once per kernel and device.
int sb_allow_smem(const void* kernel, int bytes);

// Whether a call has few enough query rows per key head for the decoding-step kernel (step_attention.cu).
bool sb_few_rows(const SbCrossAttention* g);
int sb_step_cross_attention(const SbCrossAttention* g, void* out, void* rest, float* lse, void* ws, cudaStream_t stream);
