// Shared parts of the fused cross-attention kernels (cross_attention_fwd.cu, cross_attention_bwd.cu).
//
// All query rows that read the same memory and key head are packed: row r in [0, R), R = G * rep * Tq, is token t = r % Tq of query
// head hk * rep + (r / Tq) % rep of batch row m * G + r / (Tq * rep).  A tile of 128 packed rows therefore never mixes memories,
// short queries of several heads or beams fill one tile, and the sums over shared heads and shared rows need no second pass.
#pragma once
#include "packed_math.cuh"
#include "tcgen05.cuh"
#include <cuda_fp16.h>

struct XAttnArgs {
  const void* q;                       // [B, Tq, H, D], element strides below, D contiguous
  long long q_sb, q_st, q_sh;
  const int* lengths;                  // [M] visible keys, null = Tk; clamped to [0, Tk]
  const uint8_t* mask;                 // [M, Tk] non-zero = hidden, or null
  int M, G, rep, Tq, Tk, H, Hk, D;
  int R;                               // packed rows of one (memory, key head)
  float c;                             // softmax scale * log2(e): probabilities are powers of two of c * score
  int* status;
};

namespace {

template <typename T> struct Half2;    // 16-bit types of the tensor core
template <> struct Half2<__nv_bfloat16> {
  static constexpr uint32_t KIND = 1;  // operand type field of the instruction descriptor
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
};
template <> struct Half2<__half> {
  static constexpr uint32_t KIND = 0;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 t = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
};

// D fp32, A and B of type KIND, B either K-major or MN-major, M = 128
template <typename T> constexpr uint32_t instr_desc(int n, bool b_mn) {
  return (1u << 4) | (Half2<T>::KIND << 7) | (Half2<T>::KIND << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

// `bytes` from global to shared memory, all multiples of 16
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// A operand in tensor memory (128 lanes, two 16-bit elements per column), B in shared memory
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Load and wait in one statement, so that no use of the registers can be scheduled before the wait.
__device__ __forceinline__ void tmem_load32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_load64(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
        "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// whole-warp bounded wait: the same answer in every lane, so that the .aligned instructions that follow stay converged
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* status, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, code) ? 1 : 0) != 0;
}

struct RowAt { int b, t, h; };
__device__ __forceinline__ RowAt row_at(const XAttnArgs& a, int m, int hk, int r) {
  const int x = r / a.Tq, g = x / a.rep;
  return {m * a.G + g, r - x * a.Tq, hk * a.rep + x - g * a.rep};
}

__device__ __forceinline__ int visible_keys(const XAttnArgs& a, int m) {
  if (!a.lengths) return a.Tk;
  const int n = a.lengths[m];
  return n < 0 ? 0 : (n > a.Tk ? a.Tk : n);
}

// Whether key `key` of memory m is hidden.
__device__ __forceinline__ bool hidden_key(const XAttnArgs& a, int m, int len, int key) {
  return key >= len || (a.mask && a.mask[(long long)m * a.Tk + key] != 0);
}

// By a warp: whether the mask leaves exactly one of memory m's keys.  Its softmax is then constant, and dq and dk are zero; p (dp - delta) from
// rounded p and delta would be their rounding.  Ends with the second visible key, so that only a memory that is hidden nearly wholly is read to
// its end.
__device__ __forceinline__ bool one_key_left(const XAttnArgs& a, int m, int len, int lane) {
  const uint8_t* mask = a.mask + (long long)m * a.Tk;
  int n = 0;
  for (int k0 = 0; k0 < len && n < 2; k0 += 512) {
    int mine = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int key = k0 + 32 * i + lane;
      mine += key < len && mask[key] == 0;
    }
    n += __reduce_add_sync(0xffffffffu, mine);
  }
  return n == 1;
}

// Rows of a [rows, DP] operand tile in shared memory: 64-element halves of 128-byte rows, 16-byte chunks XORed with the row (the
// 128-byte swizzle of TMA and of the matrix descriptors).
__device__ __forceinline__ uint32_t tile_addr(uint32_t base, int rows, int row, int chunk) {
  return base + (uint32_t)(chunk >> 3) * (uint32_t)(rows * 128) + (uint32_t)row * 128u + (uint32_t)(((chunk & 7) ^ (row & 7)) << 4);
}

// Element offset of this lane's packed row (row0 + lane) in a [B, Tq, H, D] tensor, -1 behind the last row.
__device__ __forceinline__ long long row_offset(const XAttnArgs& a, long long sb, long long st, long long sh, int m, int hk, int row) {
  if (row >= a.R) return -1;
  const RowAt w = row_at(a, m, hk, row);
  return w.b * sb + w.t * st + w.h * sh;
}

// A warp copies its 32 packed rows (offsets by lane, -1: zeros) into rows [quarter * 32, + 32) of a swizzled [128, DP] tile, columns
// beyond D as zeros; whole rows per instruction.
template <int DP>
__device__ __forceinline__ void load_rows(const void* src, long long off, int D, uint32_t tile, int quarter, int lane) {
  constexpr int CH = DP / 8, RPI = 32 / CH;               // 16-byte chunks of a row, rows per instruction
  const int sub = lane / CH, ch = lane % CH;
#pragma unroll 8
  for (int i = 0; i < 32; i += RPI) {
    const long long o = __shfl_sync(0xffffffffu, off, i + sub);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (o >= 0 && ch * 8 < D) v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(src) + o + ch * 8);
    st_shared_v4(tile_addr(tile, 128, quarter * 32 + i + sub, ch), v.x, v.y, v.z, v.w);
  }
}

// This lane's row of such a tile into tensor memory as an A operand: DP / 2 columns of two 16-bit elements.
template <int DP> __device__ __forceinline__ void row_to_tmem(uint32_t tile, int row, uint32_t taddr) {
#pragma unroll
  for (int h = 0; h < DP / 64; ++h) {
    uint32_t r[32];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[4 * k]), "=r"(r[4 * k + 1]), "=r"(r[4 * k + 2]), "=r"(r[4 * k + 3])
                   : "r"(tile_addr(tile, 128, row, 8 * h + k)) : "memory");
    tmem_store32(taddr + 32 * h, r);
  }
}

// What the rounding of a pair to 16 bits took away, in 16 bits again: the backward pass needs sum(do * o) to more than 16 bits, because
// it is subtracted from values of its own size.
template <typename T> __device__ __forceinline__ uint32_t out_pair(float x, float y, uint32_t& rest) {
  const uint32_t v = Half2<T>::pack(x, y);
  const float2 back = Half2<T>::unpack(v);
  rest = Half2<T>::pack(x - back.x, y - back.y);
  return v;
}

// A warp writes 64 columns (128 bytes) of its 32 rows: lane l holds row l, packed; `off` is its row's element offset, -1 for none.  The
// rows pass through 4 KB of shared memory so that an instruction writes four whole 128-byte lines; 16 bytes of 32 different rows per
// instruction cost several times as much.  `buf`: this warp's, 128-byte aligned; columns [col, col + 64) below D are written.
__device__ __forceinline__ void store_rows64(uint32_t buf, const uint32_t* packed, uint16_t* dst, long long off, int col, int D, int lane) {
#pragma unroll
  for (int k = 0; k < 8; ++k)
    st_shared_v4(buf + (uint32_t)lane * 128u + (uint32_t)((k ^ (lane & 7)) << 4), packed[4 * k], packed[4 * k + 1], packed[4 * k + 2], packed[4 * k + 3]);
  __syncwarp();
  const int sub = lane >> 3, ch = lane & 7;
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    const int row = i + sub;
    const long long o = __shfl_sync(0xffffffffu, off, row);
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(buf + (uint32_t)row * 128u + (uint32_t)((ch ^ (row & 7)) << 4)) : "memory");
    if (o >= 0 && col + ch * 8 < D) *reinterpret_cast<uint4*>(dst + o + col + ch * 8) = v;
  }
  __syncwarp();
}

// Blocks of a cluster that share one tile of results, each over its part of the summed axis: fp32 rows of DP values stand in every
// block's shared memory, 16-byte pieces XORed with the row, and block r of n adds up and writes every n-th eight columns.
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();                                              // .aligned wants whole warps, and this often stands behind a loop that lanes leave apart
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <int DP> __device__ __forceinline__ uint32_t part_addr(uint32_t base, int row, int piece) {
  return base + (uint32_t)row * (uint32_t)(DP * 4) + (uint32_t)((piece & ~7) | ((piece ^ row) & 7)) * 16u;
}
// 64 accumulator columns of this lane's row; zeros unless `have` (for the warp) and where `zero` (for the lane)
template <int DP> __device__ __forceinline__ void keep_part64(uint32_t base, int row, int col, uint32_t taddr, bool have, bool zero = false) {
  uint32_t r[64];
  if (have) {
    tmem_load64(taddr, r);
  } else {
#pragma unroll
    for (int k = 0; k < 64; ++k) r[k] = 0u;
  }
#pragma unroll
  for (int k = 0; k < 64; ++k) r[k] = zero ? 0u : r[k];
#pragma unroll
  for (int k = 0; k < 16; ++k) st_shared_v4(part_addr<DP>(base, row, col / 4 + k), r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]);
}
__device__ __forceinline__ uint32_t in_block(uint32_t addr, int rank) {
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
  return there;
}
__device__ __forceinline__ float2 load_remote2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float load_remote(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
// sum[0 .. 7] += w * eight columns of a row in block `rank`
template <int DP> __device__ __forceinline__ void add_part8(uint32_t base, int row, int c8, int rank, float w, float* sum) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(in_block(part_addr<DP>(base, row, 2 * c8 + h), rank)) : "memory");
    sum[4 * h] = fmaf(w, v.x, sum[4 * h]);
    sum[4 * h + 1] = fmaf(w, v.y, sum[4 * h + 1]);
    sum[4 * h + 2] = fmaf(w, v.z, sum[4 * h + 2]);
    sum[4 * h + 3] = fmaf(w, v.w, sum[4 * h + 3]);
  }
}

// A warp zeroes the hidden rows (bits of w[0], w[1]) of a [64, DP] tile, two a lane: a hidden infinity or NaN would turn its zero weight
// into NaN inside a matrix product.
template <int DP> __device__ __forceinline__ void clear_rows(uint32_t tile, const uint32_t* w, int lane) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if ((w[h] >> lane) & 1u) {
#pragma unroll
      for (int ch = 0; ch < DP / 8; ++ch) st_shared_v4(tile_addr(tile, 64, h * 32 + lane, ch), 0, 0, 0, 0);
    }
}

// Hidden keys as one more step of the score product: 16 elements more per row and key, the rows' being (1, 0, ...) and the keys' (0 or -inf,
// 0, ...), so that scores come out of the tensor core as they are or -inf (of 64 x 64 scores a warp, 32 packed additions and 16 loads
// from shared memory less: forward / dq of 2 x 4 x 301 queries, 1111 keys, 16 heads of 64 on 4 with a mask 46 / 58 us for 53 / 66).  Tiles without
// swizzle: 8 rows x 16 bytes side by side, the two halves of the 16 elements 128 bytes apart, groups of rows 256.
constexpr int ONES_BYTES = 128 * 32, ADDEND_BYTES = 64 * 32;
__device__ __forceinline__ uint64_t make_desc_plain(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)(128 >> 4) << 16 | (uint64_t)(256 >> 4) << 32 | (uint64_t)1 << 46;
}
// The rows' tile, and `stages` keys' tiles as zeros behind it, by `threads` threads.
template <typename T> __device__ __forceinline__ void init_addends(uint32_t addr, int stages, int thread, int threads) {
  constexpr uint32_t ONE = Half2<T>::KIND == 0 ? 0x3c00u : 0x3f80u;
  for (int i = thread; i < (ONES_BYTES + stages * ADDEND_BYTES) / 16; i += threads)
    st_shared_v4(addr + i * 16, i < ONES_BYTES / 16 && !(i & 8) ? ONE : 0u, 0u, 0u, 0u);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// by a warp, from the block's hidden bits
template <typename T> __device__ __forceinline__ void store_addends(uint32_t addr, const uint32_t* w, int lane) {
  constexpr uint32_t HIDE = Half2<T>::KIND == 0 ? 0xfc00u : 0xff80u;
#pragma unroll
  for (int h = 0; h < 2; ++h) st_shared_v4(addr + (uint32_t)((h * 4 + (lane >> 3)) * 256 + (lane & 7) * 16), (w[h] >> lane) & 1u ? HIDE : 0u, 0u, 0u, 0u);
}

}  // namespace
