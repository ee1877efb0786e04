// Host side shared by the cross-attention entry points.
#include "cross_attention_host.h"

namespace {
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) ptr = nullptr;
    return (EncodeTiledFn)ptr;
  }();
  return fn;
}
bool aligned(const void* p, long long a, long long b, long long c) { return (((uintptr_t)p) & 15) == 0 && a % 8 == 0 && b % 8 == 0 && c % 8 == 0; }
}  // namespace

int sb_xattn_args(const SbCrossAttention* g, XAttnArgs* a) {
  if (!g || !g->q || !g->k || !g->v || (g->type != 0 && g->type != 1)) return SB_BAD_ARGUMENT;
  if (g->M <= 0 || g->G <= 0 || g->rep <= 0 || g->Tq <= 0 || g->Tk <= 0 || g->Hk <= 0 || g->D <= 0 || g->D > 128 || g->D % 8) return SB_BAD_ARGUMENT;
  if (!(g->scale > 0.f) || !(g->scale < 3e38f)) return SB_BAD_ARGUMENT;
  if (!aligned(g->q, g->q_sb, g->q_st, g->q_sh) || !aligned(g->k, g->k_sb, g->k_st, g->k_sh) || !aligned(g->v, g->v_sb, g->v_st, g->v_sh))
    return SB_BAD_ARGUMENT;
  a->q = g->q;
  a->q_sb = g->q_sb; a->q_st = g->q_st; a->q_sh = g->q_sh;
  a->lengths = g->lengths; a->mask = g->mask;
  a->M = g->M; a->G = g->G; a->rep = g->rep; a->Tq = g->Tq; a->Tk = g->Tk; a->Hk = g->Hk; a->D = g->D;
  a->H = g->Hk * g->rep;
  const long long R = (long long)g->G * g->rep * g->Tq;
  if (R > 0x7fffff00ll || g->Tk > 0x7fffff00 || (long long)g->M * g->Hk > 0x7fffffffll || (long long)g->M * g->G > 0x7fffffffll) return SB_BAD_ARGUMENT;
  a->R = (int)R;
  a->c = g->scale * 1.44269504088896f;
  a->status = sb_status_ptr();
  return a->status ? 0 : -2;
}

int sb_rows_map(CUtensorMap* map, const void* ptr, int type, int D, int T, int heads, int batch, long long st, long long sh, long long sb, int box) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return -100;
  // the driver call below wants a current context, which a thread that has made no runtime call that needs one (autograd's) lacks
  static thread_local int bound = -1;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && bound != dev) e = cudaSetDevice(dev);
  if (e != cudaSuccess) return (int)e;
  bound = dev;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)T, (cuuint64_t)heads, (cuuint64_t)batch};
  // a stride that is never used (extent 1, or a broadcast of 0 over extent 1) only has to be valid
  const cuuint64_t any = (cuuint64_t)((D + 7) / 8 * 16);
  if ((T > 1 && st <= 0) || (heads > 1 && sh <= 0) || (batch > 1 && sb <= 0)) return -101;
  const cuuint64_t strides[3] = {T > 1 ? (cuuint64_t)st * 2 : any, heads > 1 ? (cuuint64_t)sh * 2 : any, batch > 1 ? (cuuint64_t)sb * 2 : any};
  const cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1}, ones[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, type == 0 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(ptr), dims, strides, boxes, ones,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -(200 + (int)r);
}

namespace {
// Clusters of n blocks of a kernel that the GPU holds at once; asked once per kernel, size and device.  (A cluster's SMs are in one part of
// the GPU, and of the parts' 16 to 20 SMs a cluster of 8 leaves some unused.)
int clusters_at_once(const void* kernel, int n, int threads, int smem) {
  struct Seen { const void* kernel; int device, n, clusters; };
  static thread_local Seen seen[64];
  static thread_local int count = 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  for (int i = 0; i < count; ++i)
    if (seen[i].kernel == kernel && seen[i].device == dev && seen[i].n == n) return seen[i].clusters;
  SbClusterLaunch l(1, n, threads, smem, 0);
  int clusters = 0;
  if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &l.config) != cudaSuccess) {
    cudaGetLastError();
    clusters = 0;
  }
  if (count < 64) seen[count++] = {kernel, dev, n, clusters};
  return clusters;
}
}  // namespace

SbTilePlan sb_plan_tiles(const void* kernel, int threads, int smem, long long tiles, int steps, int own, int join) {
  SbTilePlan plan = {tiles, 1};
  const long long sms = sb_num_sms(), left = tiles % sms;
  if (left != tiles) join += 2;                              // a launch more
  long long least = steps + own;
  for (int n = 2; n <= 8 && steps >= 2 * n && left > 0; n *= 2) {
    const int at_once = clusters_at_once(kernel, n, threads, smem);
    if (at_once <= 0) break;
    const long long cost = (left + at_once - 1) / at_once * ((steps + n - 1) / n + own + join);
    if (cost < least) {
      plan = {tiles - left, n};
      least = cost;
    }
  }
  return plan;
}

int sb_allow_smem(const void* kernel, int bytes) {
  // a handful of kernels: remembered per device, so that a launch costs no driver call
  struct Seen { const void* kernel; int device; };
  static thread_local Seen seen[64];
  static thread_local int n = 0;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  for (int i = 0; i < n; ++i)
    if (seen[i].kernel == kernel && seen[i].device == dev) return 0;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return (int)e;
  if (n < 64) seen[n++] = {kernel, dev};
  return 0;
}
