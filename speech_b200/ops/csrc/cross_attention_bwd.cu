// Fused cross attention, backward:   p = 2^(c s - lse),  dp = do v^T,  ds = p (dp - delta),  delta = sum_d do o
//   dq = scale ds k        (one CTA per 128 packed query rows, keys stream past: xattn_dq_kernel)
//   dv = p^T do, dk = scale ds^T q   (one CTA per 128 keys, packed query rows stream past: xattn_dkv_kernel)
//
// Probabilities are computed again from the scores and the row's lse, in both kernels: seven products where one kernel with shared
// sums of dq would need five, but every sum is taken by one CTA in a fixed order, so that gradients are the same every time, nothing
// is accumulated in fp32 memory and converted afterwards, and gradients of shared heads and shared rows are sums over packed rows.
//
// The products into 64 columns have a warp each that issues them: such an instruction takes the tensor core 32 cycles, and issuing it
// costs a warp twice that, so that one issuer for all of them left the tensor core idle more than half of the time.
//
// Both kernels have the roles of the forward pass otherwise.  dq: two warpgroups take blocks of 64 keys in turn; scores and dp leave tensor memory
// for registers at once, so that those of the next block are computed under this one's exponentials; q and do are A operands in tensor
// memory, because a product of 128 x 64 x 16 that reads 6 KB from shared memory takes 60 cycles, not 32.  dk / dv: tiles of 64 query rows of one head,
// transposed (lanes are keys), so that p^T and ds^T are A operands as they come out of the softmax; two pairs of warpgroups take them in
// turn, half of the columns each.  Rows come by TMA, their statistics by bulk copies, for which the dq kernel,
// which comes first and computes delta as it loads do, lays out -lse and -delta in lines of a multiple of 64 per (memory, head).
//
// Where there are fewer tiles than SMs, up to eight CTAs of a cluster share one (keys of dq, query rows of dk / dv in parts) and add their
// fp32 sums up through one another's shared memory, in a fixed order.
//
// A softmax over one key is constant: dq and dk of a memory with one visible key are multiplied by zero at the end (of its NaN and
// infinities they keep the NaN).
//
// Rounding: p and ds are rounded to the operands' 16-bit type for the products that sum them, all else is fp32.  In fp16 their range
// matters: p is multiplied by 2^12 (it is at most 1), ds by a power of two that brings the largest |do|, or a 64th of the largest
// |delta| where the values are that large, to [8, 16), and the sums are scaled back, so that neither small weights nor small upstream
// gradients fall below the type's normal range.  ds stays below its end whatever the values are: |dp| <= |do| |v| (norms), and
// |ds| = p |dp - sum p dp| <= p (1 - p) 2 max |dp| <= max |do| |v| / 2.  A kernel ahead takes the largest norm of a visible value, and where
// sqrt(D) max|v| exceeds 4096 the peak of do counts that many times as much: ds then ends below 16 * 2048.  (Not needed for bf16; in fp16 it
// reads the values once more: 4 us of 197 for forward and backward of 12 x 301 queries, 3 x 1111 keys, 16 heads on 4 of 64, 8 of 575 for 4 x 1024
// queries, 7500 keys, 8 heads of 128.)
#include "cross_attention.cuh"
#include "cross_attention_host.h"

namespace {

constexpr int DKV_THREADS = 640;       // 20 warps of 96 registers
// What a CTA takes besides its blocks or steps, in those; a join takes half of it.  [dq, 100 queries, 8 heads of 128, 1 / 2 / 4 / 8 CTAs a
// tile: 74 / 47 / 33 / 27 us for 7500 keys, 25 / 23 / 18 / 18 for 1500; dk / dv, 5 x 1500 queries against 100 keys: 102 / 59 / 37 / 29 us]
constexpr int DQ_OWN_BLOCKS = 10, DKV_OWN_STEPS = 8;
template <typename T> constexpr float p_shift() { return Half2<T>::KIND == 0 ? 12.f : 0.f; }

struct BwdArgs {
  const uint16_t* dout;               // contiguous [B, Tq, H, D]
  const uint16_t *out, *rest;         // the forward pass's result and what its rounding took away
  const float* lse;                   // [M * Hk, R]
  float *nlse, *ndelta;               // [M * Hk, G * rep, Tqp]: -lse (-inf behind the last row, too) and -delta (0 there)
  int Tqp;                            // Tq rounded up to 64
  float* peak;                        // fp16: what ds_scale() takes, of every block of the dq kernel
  float* norms;                       // fp16: the largest norm of a visible value, of every NORM_KEYS keys of a (memory, key head)
  int tiles;                          // its blocks of a (memory, key head)
  float scale;
};

// Power of two that brings the peak of a (memory, key head) to [8, 16); 1 for bf16, whose range needs none.  The peak is the largest
// |do| (times sqrt(D) max|v| / 4096 where that is above one), or |delta| / 64.
template <typename T> __device__ __forceinline__ float ds_scale(float peak) {
  if (Half2<T>::KIND != 0 || !(peak > 0.f) || !(peak < 3e38f)) return 1.f;
  return __int_as_float((127 + 3 - ((__float_as_int(fmaxf(peak, 1e-8f)) >> 23) - 127)) << 23);      // |do| of fp16 is at least 2^-24
}

// Few keys a block: it is the latency of its loads that counts (256 keys: 9 us for 64 at 3 x 1111 keys, 4 heads of 64).
constexpr int NORM_KEYS = 64;
__host__ __device__ inline int norm_parts(int Tk) { return (Tk + NORM_KEYS - 1) / NORM_KEYS; }
template <int DP>
__global__ void __launch_bounds__(256) xattn_norms_kernel(const XAttnArgs a, const __half* __restrict__ v, const long long sb, const long long st,
                                                          const long long sh, float* __restrict__ norms, const int parts) {
  constexpr int CH = DP / 8;
  const int unit = blockIdx.x / parts, key0 = (blockIdx.x - unit * parts) * NORM_KEYS, m = unit / a.Hk, hk = unit % a.Hk;
  const int len = visible_keys(a, m), sub = threadIdx.x / CH, ch = threadIdx.x % CH;
  const __half* at = v + m * sb + hk * sh + ch * 8;
  float top = 0.f;
#pragma unroll
  for (int r = sub; r < NORM_KEYS; r += 256 / CH) {
    const int key = key0 + r;
    const bool in = ch * 8 < a.D && key < len;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (in) x = *reinterpret_cast<const uint4*>(at + key * st);
    if (a.mask && in && a.mask[(long long)m * a.Tk + key]) x = make_uint4(0, 0, 0, 0);      // read beside its value, not before
    const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = Half2<__half>::unpack(xs[k]);
      sum += f.x * f.x + f.y * f.y;
    }
#pragma unroll
    for (int s = CH / 2; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    top = fmaxf(top, sum);
  }
  __shared__ float red[8];
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, red[i]);
    norms[blockIdx.x] = sqrtf(top);
  }
}

// By a warp: what the largest |do| counts for the values' sake.
template <typename T> __device__ __forceinline__ float value_factor(const XAttnArgs& a, const BwdArgs& b, int unit, int lane) {
  if (Half2<T>::KIND != 0) return 1.f;
  const int parts = norm_parts(a.Tk);
  float top = 0.f;
  for (int i = lane; i < parts; i += 32) top = fmaxf(top, b.norms[(long long)unit * parts + i]);
  return fmaxf(1.f, warp_max(top) * sqrtf((float)a.D) * (1.f / 4096.f));
}

// A warp's 32 rows of do into a swizzled tile (as load_rows), with sum(do * (out + rest)) of this lane's row and the peak of all.
template <typename T, int DP>
__device__ __forceinline__ void load_do_rows(const BwdArgs& b, long long off, int D, uint32_t tile, int quarter, int lane, float& delta, float& peak,
                                             float factor) {
  constexpr int CH = DP / 8, RPI = 32 / CH;
  const int sub = lane / CH, ch = lane % CH;
  delta = peak = 0.f;
#pragma unroll 4
  for (int i = 0; i < 32; i += RPI) {
    const long long o = __shfl_sync(0xffffffffu, off, i + sub);
    uint4 x = make_uint4(0, 0, 0, 0), y = x, z = x;
    if (o >= 0 && ch * 8 < D) {
      x = *reinterpret_cast<const uint4*>(b.dout + o + ch * 8);
      y = *reinterpret_cast<const uint4*>(b.out + o + ch * 8);
      z = *reinterpret_cast<const uint4*>(b.rest + o + ch * 8);
    }
    st_shared_v4(tile_addr(tile, 128, quarter * 32 + i + sub, ch), x.x, x.y, x.z, x.w);
    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w}, zs[4] = {z.x, z.y, z.z, z.w};
    float d = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = Half2<T>::unpack(xs[k]), e = Half2<T>::unpack(ys[k]), c = Half2<T>::unpack(zs[k]);
      d += f.x * (e.x + c.x) + f.y * (e.y + c.y);
      if (Half2<T>::KIND == 0) peak = fmaxf(peak, fmaxf(fabsf(f.x), fabsf(f.y)));
    }
#pragma unroll
    for (int s = CH / 2; s > 0; s >>= 1) d += __shfl_xor_sync(0xffffffffu, d, s);
    const float mine = __shfl_sync(0xffffffffu, d, ((lane - i) & (RPI - 1)) * CH);
    if (lane >= i && lane < i + RPI) delta = mine;
  }
  if (Half2<T>::KIND == 0) peak = warp_max(fmaxf(peak * factor, fabsf(delta) * (1.f / 64.f)));
}

// Eight columns of a row from all blocks of the cluster, in turn, times f, rounded and written.
template <typename T, int DP> __device__ __forceinline__ void join_parts8(uint32_t base, int row, int c8, int splits, float f, uint16_t* dst) {
  float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < splits; ++i) add_part8<DP>(base, row, c8, i, 1.f, o);
  *reinterpret_cast<uint4*>(dst) = make_uint4(Half2<T>::pack(o[0] * f, o[1] * f), Half2<T>::pack(o[2] * f, o[3] * f), Half2<T>::pack(o[4] * f, o[5] * f),
                                              Half2<T>::pack(o[6] * f, o[7] * f));
}

// 64 accumulator columns of a warp's 32 rows, times f, rounded and written; zeros unless `have`, and in the lanes' rows with `zero`.
template <typename T>
__device__ __forceinline__ void store_acc64(uint32_t buf, uint32_t taddr, bool have, float f, uint16_t* dst, long long off, int col, int D, int lane,
                                            bool zero = false) {
  uint32_t r[64], v[32];
  if (have) {
    tmem_load64(taddr, r);
  } else {
#pragma unroll
    for (int k = 0; k < 64; ++k) r[k] = 0u;
  }
#pragma unroll
  for (int k = 0; k < 32; ++k) v[k] = zero ? 0u : Half2<T>::pack(__uint_as_float(r[2 * k]) * f, __uint_as_float(r[2 * k + 1]) * f);
  store_rows64(buf, v, dst, off, col, D, lane);
}

// ------------------------------------------------------------------------------------------------ dq
template <int DP> struct DqSmem {
  static constexpr int BN = 64;
  static constexpr int STAGES = 5;
  static constexpr int ROWS = 128 * DP * 2, KEYS = BN * DP * 2;
  static constexpr int DO0 = ROWS, KV0 = 2 * ROWS, BAR = KV0 + STAGES * 2 * KEYS;
  static constexpr int ONES0 = 0, ADD0 = ONES0 + ONES_BYTES;        // where the queries were, once they are in tensor memory
  static constexpr int BYTES = BAR + 768 + 1024;
  static_assert(ADD0 + STAGES * ADDEND_BYTES <= ROWS, "");
  // tensor memory: dq, q, do, scores of even and odd blocks, dp, ds of even and odd blocks
  static constexpr int Q_COL = DP, DO_COL = DP + DP / 2, S_COL = 2 * DP, DP_COL = S_COL + 128, DS_COL = DP_COL + 64;
};
constexpr int DQ_THREADS = 384;

template <typename T, int DP>
__global__ void __launch_bounds__(DQ_THREADS, 1)
xattn_dq_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const XAttnArgs a, const BwdArgs b,
                uint16_t* __restrict__ dq, const long long tile0, const int splits) {
  using S = DqSmem<DP>;
  constexpr int BN = S::BN, HALVES = DP / 64;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bars = base + S::BAR;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto kv_full = [&](int s) { return bars + 8u * s; };
  auto kv_empty = [&](int s) { return bars + 8u * (5 + s); };
  auto s_full = [&](int u) { return bars + 8u * (10 + u); };
  auto s_read = [&](int u) { return bars + 8u * (12 + u); };
  auto ds_full = [&](int u) { return bars + 8u * (14 + u); };
  auto ds_read = [&](int u) { return bars + 8u * (16 + u); };
  auto dp_full = [&](int u) { return bars + 8u * (18 + u); };     // one per warpgroup: each sees every other block only
  auto kv_clean = [&](int s) { return bars + 8u * (24 + s); };
  const uint32_t dp_read = bars + 8u * 20, dq_full = bars + 8u * 21, rows_ready = bars + 8u * 22, tmem_slot = bars + 8u * 23;
  const uint32_t seen_slot = bars + 8u * 29;               // whether the mask leaves any of these keys
  const uint32_t one_slot = seen_slot + 4;                 // whether just one of the memory's is visible
  const uint32_t stats = bars + 240u;                      // -delta of the tile's rows, peaks of four warps

  const int tiles = b.tiles;
  const int local = blockIdx.x / splits, rank = blockIdx.x - local * splits;      // block `rank` of a cluster takes its part of the keys
  const int index = (int)tile0 + local;
  const int unit = index / tiles, m = unit / a.Hk, hk = unit % a.Hk;
  const int row0 = (index - unit * tiles) * 128;
  const int len = visible_keys(a, m);
  const int blocks = (len + BN - 1) / BN;
  const int share = (blocks + splits - 1) / splits, first = rank * share * BN;
  const int nt = dq || blocks == 1 ? min(share, max(0, blocks - rank * share)) : 0;      // without dq only the statistics are wanted, for which one block refines delta
  const bool hide = a.mask != nullptr;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) { mbar_init(kv_full(s), 1); mbar_init(kv_clean(s), 1); mbar_init(kv_empty(s), 1); }
    for (int u = 0; u < 2; ++u) { mbar_init(s_full(u), 1); mbar_init(s_read(u), 4); mbar_init(ds_full(u), 4); mbar_init(ds_read(u), 1); mbar_init(dp_full(u), 1); }
    mbar_init(dp_read, 4);
    mbar_init(dq_full, 1);
    mbar_init(rows_ready, 8);
    if (!hide) asm volatile("st.shared.u32 [%0], %1;" ::"r"(one_slot), "r"((uint32_t)(len == 1)) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tmem_slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot) : "memory");

  if (warp == 0) {
    // loads, up to STAGES - 2 blocks ahead, so that clearing runs two blocks ahead of dq; hidden keys' rows are cleared as they land (their
    // ds is zero, and zero times NaN is not)
    auto load = [&](int j) {
      const int s = j % S::STAGES;
      if (!warp_wait(kv_empty(s), ((uint32_t)(j / S::STAGES) & 1u) ^ 1u, a.status, SB_TIMEOUT_SMEM_EMPTY)) return false;
      if (elect_one()) {
        const uint32_t kb = base + S::KV0 + s * 2 * S::KEYS;
        mbar_expect_tx(kv_full(s), 2 * S::KEYS);
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          tma_load_4d(kb + h * (BN * 128), &map_k, kv_full(s), h * 64, first + j * BN, hk, m);
          tma_load_4d(kb + S::KEYS + h * (BN * 128), &map_v, kv_full(s), h * 64, first + j * BN, hk, m);
        }
      }
      __syncwarp();
      return true;
    };
    int issued = 0;
    bool ok = true;
    for (; issued < nt && issued < S::STAGES - 2 && ok; ++issued) ok = load(issued);
    bool hid[2] = {hidden_key(a, m, len, first + lane), hidden_key(a, m, len, first + 32 + lane)};      // this lane's keys of block j, read a block ahead
    if (nt > 0 && ok && (hide || first + nt * BN > len)) {
      ok = warp_wait(rows_ready, 0, a.status, SB_TIMEOUT_SMEM_FULL);
      if (ok) init_addends<T>(base + S::ONES0, S::STAGES, lane, 32);
      __syncwarp();
    }
    bool seen = false;
    for (int j = 0; j < nt && ok; ++j) {
      const int s = j % S::STAGES;
      const bool some = hide || first + (j + 1) * BN > len;
      uint32_t w[2] = {0, 0};
      if (some) {
#pragma unroll
        for (int i = 0; i < 2; ++i) w[i] = __ballot_sync(0xffffffffu, hid[i]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) hid[i] = hidden_key(a, m, len, first + (j + 1) * BN + 32 * i + lane);
      ok = warp_wait(kv_full(s), (uint32_t)(j / S::STAGES) & 1u, a.status, SB_TIMEOUT_SMEM_FULL);
      if (!ok) break;
      if (some) {
        clear_rows<DP>(base + S::KV0 + s * 2 * S::KEYS, w, lane);
        clear_rows<DP>(base + S::KV0 + s * 2 * S::KEYS + S::KEYS, w, lane);
        store_addends<T>(base + S::ADD0 + s * ADDEND_BYTES, w, lane);
        seen |= (w[0] & w[1]) != 0xffffffffu;
        if (j == nt - 1 && lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(seen_slot), "r"((uint32_t)seen) : "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(kv_clean(s));
      if (issued < nt) {
        ok = load(issued);
        if (ok) ++issued;
      }
    }
    // no copy may be in flight when the block ends (none is, unless a wait gave up)
    for (int i = issued > S::STAGES ? issued - S::STAGES : 0; i < issued; ++i)
      warp_wait(kv_full(i % S::STAGES), (uint32_t)(i / S::STAGES) & 1u, a.status, SB_TIMEOUT_SMEM_FULL);
  } else if (warp == 1 || warp == 3) {
    // s = q k^T (warp 1) into the columns of block j & 1, dp = do v^T (warp 3) into its only ones: each as soon as the columns have been
    // read, which happens right before a warpgroup starts on them
    const bool second = warp == 3;
    constexpr uint32_t idesc_s = instr_desc<T>(BN, false);
    const uint32_t rows = tmem + (second ? S::DO_COL : S::Q_COL);
    const uint64_t kd = make_desc(base + S::KV0 + (second ? S::KEYS : 0), 16, 1024);
    bool ok = nt > 0 && warp_wait(rows_ready, 0, a.status, SB_TIMEOUT_SMEM_FULL);
    int s = 0;
    uint32_t ph = 0;
    for (int j = 0; j < nt && ok; ++j) {
      ok = warp_wait(hide || first + (j + 1) * BN > len ? kv_clean(s) : kv_full(s), ph, a.status, SB_TIMEOUT_SMEM_FULL) &&
           (second ? warp_wait(dp_read, ((uint32_t)j & 1u) ^ 1u, a.status, SB_TIMEOUT_TMEM_EMPTY)
                   : warp_wait(s_read(j & 1), ((uint32_t)(j >> 1) & 1u) ^ 1u, a.status, SB_TIMEOUT_TMEM_EMPTY));
      if (!ok) break;
      tc_fence_after();
      const uint64_t st = (uint64_t)((s * 2 * S::KEYS) >> 4);
      const uint32_t d = tmem + (second ? S::DP_COL : S::S_COL + (j & 1) * 64);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
          umma_ts(d, rows + kk * 8, kd + st + (uint64_t)(((kk >> 2) * (BN * 128) + (kk & 3) * 32) >> 4), idesc_s, kk > 0);
        if (!second && (hide || first + (j + 1) * BN > len))
          umma_bf16(d, make_desc_plain(base + S::ONES0), make_desc_plain(base + S::ADD0 + s * ADDEND_BYTES), idesc_s, 1);
        umma_commit(second ? dp_full(j & 1) : s_full(j & 1));
      }
      __syncwarp();
      if (++s == S::STAGES) { s = 0; ph ^= 1u; }
    }
  } else if (warp == 2) {
    // dq += ds k
    if (hide) {
      const bool one = one_key_left(a, m, len, lane);
      if (lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(one_slot), "r"((uint32_t)one) : "memory");
      __syncwarp();
      asm volatile("bar.arrive 2, 288;" ::: "memory");
    }
    constexpr uint32_t idesc_o = instr_desc<T>(DP, true);
    const uint64_t kn = make_desc(base + S::KV0, BN * 128, 1024);
    bool ok = true;
    int s = 0;
    for (int j = 0; j < nt && ok; ++j) {
      ok = warp_wait(ds_full(j & 1), (uint32_t)(j >> 1) & 1u, a.status, SB_TIMEOUT_TMEM_EMPTY);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk)
          umma_ts(tmem, tmem + S::DS_COL + (j & 1) * 32 + kk * 8, kn + (uint64_t)((s * 2 * S::KEYS + kk * 2048) >> 4), idesc_o, (j > 0) | (kk > 0));
        umma_commit(ds_read(j & 1));
        umma_commit(kv_empty(s));
        if (j == nt - 1) umma_commit(dq_full);
      }
      __syncwarp();
      if (++s == S::STAGES) s = 0;
    }
  } else {
    // two warpgroups take even and odd key blocks
    const int wg = (warp - 4) >> 2, quarter = warp & 3;
    const int row = row0 + quarter * 32 + lane;
    const bool valid = row < a.R;
    const int line = row / a.Tq, t = row - line * a.Tq;
    const long long stat = valid ? ((long long)unit * (a.G * a.rep) + line) * b.Tqp + t : 0;
    const float nlse = valid ? -b.lse[(long long)unit * a.R + row] : -INFINITY;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_addr = lane_base + S::S_COL + wg * 64, dp_addr = lane_base + S::DP_COL, ds_addr = lane_base + S::DS_COL + wg * 32;
    bool ok = true;
    // q by the first, do (and with it delta) by the second, through shared memory into tensor memory
    const uint32_t tile = base + wg * S::DO0, stat_row = stats + (uint32_t)(quarter * 32 + lane) * 4u;
    const long long st = (long long)a.H * a.D;
    if (wg == 0) {
      load_rows<DP>(a.q, row_offset(a, a.q_sb, a.q_st, a.q_sh, m, hk, row), a.D, tile, quarter, lane);
    } else {
      float delta, peak;
      load_do_rows<T, DP>(b, row_offset(a, st * a.Tq, st, a.D, m, hk, row), a.D, tile, quarter, lane, delta, peak, value_factor<T>(a, b, unit, lane));
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(stat_row), "f"(-delta) : "memory");
      if (lane == 0) asm volatile("st.shared.f32 [%0], %1;" ::"r"(stats + (128 + quarter) * 4), "f"(peak) : "memory");
      if (valid && rank == 0) {
        b.nlse[stat] = nlse;
        if (blocks != 1) b.ndelta[stat] = -delta;
        if (t == a.Tq - 1)                                   // the line's end, which the copies of the dk / dv kernel read
          for (int x = 1; x < b.Tqp - t; ++x) {
            b.nlse[stat + x] = -INFINITY;
            b.ndelta[stat + x] = 0.f;
          }
      }
    }
    __syncwarp();                                            // lanes wrote statistics by themselves
    if (nt > 0) {
      row_to_tmem<DP>(tile, quarter * 32 + lane, lane_base + (wg ? S::DO_COL : S::Q_COL));
      tmem_store_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(rows_ready);
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");           // both warpgroups: the statistics in shared memory
    float ndelta, p4[4];
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(ndelta) : "r"(stat_row) : "memory");
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(p4[i]) : "r"(stats + (128 + i) * 4) : "memory");
    const float peak = fmaxf(fmaxf(p4[0], p4[1]), fmaxf(p4[2], p4[3])), dsf = ds_scale<T>(peak);
    if (Half2<T>::KIND == 0 && warp == 4 && lane == 0 && rank == 0) b.peak[index] = peak;
    const uint64_t c2 = pair(a.c, a.c), nl2 = pair(nlse, nlse), f2 = pair(dsf, dsf);
    uint32_t ph = 0;
    for (int j = wg; j < nt; j += 2) {
      uint32_t r[64], g[64];
      ok = warp_wait(s_full(wg), ph, a.status, SB_TIMEOUT_TMEM_FULL);
      if (!ok) break;
      tc_fence_after();
      tmem_load64(s_addr, r);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_read(wg));
      ok = warp_wait(dp_full(wg), ph, a.status, SB_TIMEOUT_TMEM_FULL);
      if (!ok) break;
      tc_fence_after();
      tmem_load64(dp_addr, g);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(dp_read);
      // Waited for here and not where ds is stored: the branches keep the arithmetic below from being scheduled before the arrivals above,
      // which nothing in this warp depends on but the next products do (1480 -> 1200 cycles a block).
      if (j >= 2) {
        ok = warp_wait(ds_read(wg), ph ^ 1u, a.status, SB_TIMEOUT_TMEM_FULL);
        if (!ok) break;
        tc_fence_after();
      }
#pragma unroll
      for (int k = 0; k < 64; k += 2) {                    // p over s
        float x, y;
        split(fma2(pair(r[k], r[k + 1]), c2, nl2), x, y);
        r[k] = __float_as_uint(ex2(x));
        r[k + 1] = __float_as_uint(ex2(y));
      }
      if (blocks == 1) {
        // all keys are in this block: delta = sum p dp from the values that it is subtracted from, instead of the rounded output
        uint64_t d2[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < 64; k += 2) d2[(k >> 1) & 1] = fma2(pair(r[k], r[k + 1]), pair(g[k], g[k + 1]), d2[(k >> 1) & 1]);
        float x, y;
        split(add2(d2[0], d2[1]), x, y);
        ndelta = -(x + y);
        if (valid) b.ndelta[stat] = ndelta;
        __syncwarp();
      }
      const uint64_t nd2 = pair(ndelta, ndelta);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t o[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const int e = 32 * i + 2 * k;
          uint64_t v = mul2(pair(r[e], r[e + 1]), add2(pair(g[e], g[e + 1]), nd2));
          if (Half2<T>::KIND == 0) v = mul2(v, f2);
          float x, y;
          split(v, x, y);
          o[k] = Half2<T>::pack(x, y);
        }
        tmem_store16(ds_addr + 16 * i, o);
      }
      tmem_store_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full(wg));
      ph ^= 1u;
    }
    if (nt > 0 && ok) ok = warp_wait(dq_full, 0, a.status, SB_TIMEOUT_TMEM_FULL);
    tc_fence_after();
    if (hide && nt > 0 && ok) {                              // zero where the mask leaves nothing, whatever the query holds
      uint32_t seen = 1;
      ok = warp_wait(kv_clean((nt - 1) % S::STAGES), (uint32_t)((nt - 1) / S::STAGES) & 1u, a.status, SB_TIMEOUT_SMEM_FULL);
      if (ok) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(seen) : "r"(seen_slot) : "memory");
      ok = ok && seen;
    }
    if (hide) asm volatile("bar.sync 2, 288;" ::: "memory");      // with warp 2
    uint32_t one;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(one) : "r"(one_slot) : "memory");
    if (splits > 1) {
      if (wg < DP / 64) keep_part64<DP>(base, quarter * 32 + lane, 64 * wg, lane_base + 64 * wg, nt > 0 && ok);
    } else if (dq && wg < DP / 64) {                       // 64 columns a warpgroup
      const long long off = row_offset(a, (long long)a.Tq * a.H * a.D, (long long)a.H * a.D, a.D, m, hk, row);
      store_acc64<T>(base + (wg * 4 + quarter) * 4096, lane_base + 64 * wg, nt > 0 && ok, one ? 0.f : b.scale / dsf, dq, off, 64 * wg, a.D, lane);
    }
  }
  if (splits > 1) {                                        // only with dq
    __syncthreads();
    cluster_sync();
    float peak = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float p;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(p) : "r"(stats + (128 + i) * 4) : "memory");
      peak = fmaxf(peak, p);
    }
    uint32_t one;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(one) : "r"(one_slot) : "memory");
    const float f = one ? 0.f : b.scale / ds_scale<T>(peak);
    constexpr int CH = DP / 8;
    for (int x = rank * DQ_THREADS + threadIdx.x; x < 128 * CH; x += splits * DQ_THREADS) {
      const int r = x / CH, c8 = x % CH;
      if (row0 + r >= a.R || c8 * 8 >= a.D) continue;
      join_parts8<T, DP>(base, r, c8, splits, f, dq + row_offset(a, (long long)a.Tq * a.H * a.D, (long long)a.H * a.D, a.D, m, hk, row0 + r) + c8 * 8);
    }
    cluster_sync();                                          // the others may still read this block's part
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// ------------------------------------------------------------------------------------------------ dk, dv
template <int DP> struct DkvSmem {
  static constexpr int BQ = 64;                            // query rows of a step
  static constexpr int STAGES = 4;
  static constexpr int KEYS = 128 * DP * 2, ROWS = BQ * DP * 2, STAT = 2 * BQ * 4;
  static constexpr int Q0 = 2 * KEYS, STAT0 = Q0 + STAGES * 2 * ROWS, BAR = STAT0 + STAGES * STAT;
  static constexpr int BYTES = BAR + 256 + 1024;
  // tensor memory: dv, dk, k (and v for DP = 64, where there is room) as A operands, scores, dp, p and ds
  static constexpr bool V_TMEM = DP == 64;
  static constexpr int DK_COL = DP, K_COL = 2 * DP, V_COL = K_COL + DP / 2, S_COL = V_COL + (V_TMEM ? DP / 2 : 0), DP_COL = S_COL + 64, P_COL = DP_COL + 64,
                       DS_COL = P_COL + 32;
};

template <typename T, int DP>
__global__ void __launch_bounds__(DKV_THREADS, 1)
xattn_dkv_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_q,
                 const __grid_constant__ CUtensorMap map_do, const XAttnArgs a, const BwdArgs b, uint16_t* __restrict__ dk, uint16_t* __restrict__ dv,
                 const long long tile0, const int splits) {
  using S = DkvSmem<DP>;
  constexpr int BQ = S::BQ, HALVES = DP / 64;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bars = base + S::BAR;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto q_full = [&](int s) { return bars + 8u * s; };
  auto q_empty = [&](int s) { return bars + 8u * (4 + s); };
  auto s_full = [&](int u) { return bars + 8u * (8 + u); };           // one per pair of warpgroups: each sees every other step only
  auto dp_full = [&](int u) { return bars + 8u * (10 + u); };
  auto p_full = [&](int u) { return bars + 8u * (12 + u); };
  auto p_read = [&](int u) { return bars + 8u * (14 + u); };
  const uint32_t s_read = bars + 8u * 16, dp_read = bars + 8u * 17, kv_full = bars + 8u * 18, kv_tmem = bars + 8u * 19, d_full = bars + 8u * 20,
                 tmem_slot = bars + 8u * 21, scale_slot = tmem_slot + 4;
  const uint32_t one_slot = bars + 8u * 22;                // whether just one of the memory's keys is visible

  const int ktiles = (a.Tk + 127) / 128;
  const int local = blockIdx.x / splits, rank = blockIdx.x - local * splits;      // block `rank` of a cluster takes its part of the rows
  const int index = (int)tile0 + local;
  const int unit = index / ktiles, m = unit / a.Hk, hk = unit % a.Hk;
  const int key0 = (index - unit * ktiles) * 128;
  const int len = visible_keys(a, m);
  const int segs = a.G * a.rep, lines = b.Tqp / BQ;        // (row, head) pairs that read these keys, steps of each
  const int share = (segs * lines + splits - 1) / splits, step0 = rank * share;
  const int nq = key0 < len ? min(share, max(0, segs * lines - step0)) : 0;        // 0: nothing is visible here, gradients are zero

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) { mbar_init(q_full(s), 1); mbar_init(q_empty(s), 1); }
    for (int u = 0; u < 2; ++u) { mbar_init(s_full(u), 1); mbar_init(dp_full(u), 1); mbar_init(p_full(u), 8); mbar_init(p_read(u), 1); }
    mbar_init(s_read, 8);
    mbar_init(dp_read, 8);
    mbar_init(kv_full, 1);
    mbar_init(kv_tmem, S::V_TMEM ? 8 : 4);
    mbar_init(d_full, 1);
    if (!a.mask) asm volatile("st.shared.u32 [%0], %1;" ::"r"(one_slot), "r"((uint32_t)(len == 1)) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tmem_slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 2) {
    float peak = 0.f;
    if (Half2<T>::KIND == 0)
      for (int i = lane; i < b.tiles; i += 32) peak = fmaxf(peak, b.peak[(long long)unit * b.tiles + i]);
    const float f = ds_scale<T>(warp_max(peak));
    if (lane == 0) asm volatile("st.shared.f32 [%0], %1;" ::"r"(scale_slot), "f"(f) : "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot) : "memory");

  if (warp == 0) {
    // ---------------------------------------------------------------- loads
    if (nq > 0 && elect_one()) {
      mbar_expect_tx(kv_full, 2 * S::KEYS);
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
#pragma unroll
        for (int r = 0; r < 128; r += 64) {                  // the dq kernel's boxes of 64 rows, two of them
          tma_load_4d(base + h * 16384 + r * 128, &map_k, kv_full, h * 64, key0 + r, hk, m);
          tma_load_4d(base + S::KEYS + h * 16384 + r * 128, &map_v, kv_full, h * 64, key0 + r, hk, m);
        }
      }
    }
    __syncwarp();
    const int seg = step0 / lines;
    // step step0 + i: rows t0 .. of head hk * rep + head of batch row m * G + g
    int s = 0, issued = 0, t0 = (step0 - seg * lines) * BQ, g = seg / a.rep, head = seg - g * a.rep;
    uint32_t ph = 0;
    for (int i = 0; i < nq; ++i) {
      if (!warp_wait(q_empty(s), ph ^ 1u, a.status, SB_TIMEOUT_SMEM_EMPTY)) break;
      if (elect_one()) {
        const uint32_t qb = base + S::Q0 + s * 2 * S::ROWS, st = base + S::STAT0 + s * S::STAT;
        const long long line = ((long long)unit * segs + g * a.rep + head) * b.Tqp + t0;
        mbar_expect_tx(q_full(s), 2 * S::ROWS + S::STAT);
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          tma_load_4d(qb + h * (BQ * 128), &map_q, q_full(s), h * 64, t0, hk * a.rep + head, m * a.G + g);
          tma_load_4d(qb + S::ROWS + h * (BQ * 128), &map_do, q_full(s), h * 64, t0, hk * a.rep + head, m * a.G + g);
        }
        bulk_load(st, b.nlse + line, BQ * 4, q_full(s));
        bulk_load(st + BQ * 4, b.ndelta + line, BQ * 4, q_full(s));
      }
      __syncwarp();
      issued = i + 1;
      if (++s == S::STAGES) { s = 0; ph ^= 1u; }
      t0 += BQ;
      if (t0 >= a.Tq) {
        t0 = 0;
        if (++head == a.rep) { head = 0; ++g; }
      }
    }
    if (nq > 0) warp_wait(kv_full, 0, a.status, SB_TIMEOUT_SMEM_FULL);
    for (int i = issued > S::STAGES ? issued - S::STAGES : 0; i < issued; ++i)
      warp_wait(q_full(i % S::STAGES), (uint32_t)(i / S::STAGES) & 1u, a.status, SB_TIMEOUT_SMEM_FULL);
  } else if (warp == 1 || warp == 2) {
    // ---------------------------------------------------------------- s^T = k q^T (warp 1), dp^T = v do^T (warp 2) of every step, each as soon
    // as its columns have been read
    const bool second = warp == 2;
    constexpr uint32_t idesc_s = instr_desc<T>(BQ, false);
    const uint64_t vd = make_desc(base + S::KEYS, 16, 1024), qd = make_desc(base + S::Q0 + (second ? S::ROWS : 0), 16, 1024);
    const uint32_t d = tmem + (second ? S::DP_COL : S::S_COL), keys = tmem + (second ? S::V_COL : S::K_COL);
    bool ok = nq > 0 && warp_wait(second && !S::V_TMEM ? kv_full : kv_tmem, 0, a.status, SB_TIMEOUT_SMEM_FULL);
    int s = 0;
    uint32_t ph = 0;
    for (int i = 0; i < nq && ok; ++i) {
      ok = warp_wait(q_full(s), ph, a.status, SB_TIMEOUT_SMEM_FULL) &&
           warp_wait(second ? dp_read : s_read, ((uint32_t)i & 1u) ^ 1u, a.status, SB_TIMEOUT_TMEM_EMPTY);
      if (!ok) break;
      tc_fence_after();
      const uint64_t st = (uint64_t)((s * 2 * S::ROWS) >> 4);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint64_t ko = (uint64_t)(((kk >> 2) * 16384 + (kk & 3) * 32) >> 4), ro = (uint64_t)(((kk >> 2) * (BQ * 128) + (kk & 3) * 32) >> 4);
          if (second && !S::V_TMEM) umma_bf16(d, vd + ko, qd + st + ro, idesc_s, kk > 0);
          else umma_ts(d, keys + kk * 8, qd + st + ro, idesc_s, kk > 0);
        }
        umma_commit(second ? dp_full(i & 1) : s_full(i & 1));
      }
      __syncwarp();
      if (++s == S::STAGES) { s = 0; ph ^= 1u; }
    }
  } else if (warp == 3) {
    // ---------------------------------------------------------------- dv += p^T do, dk += ds^T q
    if (a.mask) {
      const bool one = one_key_left(a, m, len, lane);
      if (lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(one_slot), "r"((uint32_t)one) : "memory");
      __syncwarp();
      asm volatile("bar.arrive 1, 544;" ::: "memory");
    }
    constexpr uint32_t idesc_o = instr_desc<T>(DP, true);
    const uint64_t qn = make_desc(base + S::Q0, BQ * 128, 1024);
    bool ok = true;
    int s = 0;
    for (int i = 0; i < nq && ok; ++i) {
      ok = warp_wait(p_full(i & 1), (uint32_t)(i >> 1) & 1u, a.status, SB_TIMEOUT_TMEM_EMPTY);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t st = (uint64_t)((s * 2 * S::ROWS) >> 4);
#pragma unroll
        for (int kk = 0; kk < BQ / 16; ++kk)
          umma_ts(tmem, tmem + S::P_COL + kk * 8, qn + st + (uint64_t)((S::ROWS + kk * 2048) >> 4), idesc_o, (i > 0) | (kk > 0));
#pragma unroll
        for (int kk = 0; kk < BQ / 16; ++kk)
          umma_ts(tmem + S::DK_COL, tmem + S::DS_COL + kk * 8, qn + st + (uint64_t)((kk * 2048) >> 4), idesc_o, (i > 0) | (kk > 0));
        umma_commit(p_read(i & 1));
        umma_commit(q_empty(s));
        if (i == nq - 1) umma_commit(d_full);
      }
      __syncwarp();
      if (++s == S::STAGES) s = 0;
    }
  } else {
    // ---------------------------------------------------------------- p^T and ds^T; lanes are keys
    const int u = (warp - 4) >> 3, half = ((warp - 4) >> 2) & 1, quarter = warp & 3;
    const int key = key0 + quarter * 32 + lane;
    bool ok = true;
    float dsf;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(dsf) : "r"(scale_slot) : "memory");
    const bool hidden = key >= len || (a.mask && a.mask[(long long)m * a.Tk + key] != 0);
    const bool some_hidden = __any_sync(0xffffffffu, hidden);
    const float k_ds = dsf * ex2(-p_shift<T>());
    const uint64_t c2 = pair(a.c, a.c), shift2 = pair(p_shift<T>(), p_shift<T>()), f2 = pair(k_ds, k_ds);
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
    if (nq > 0 && u == 0 && (half == 0 || S::V_TMEM)) {      // keys (and values) into tensor memory, by the first warpgroups
      ok = warp_wait(kv_full, 0, a.status, SB_TIMEOUT_SMEM_FULL);
      row_to_tmem<DP>(base + half * S::KEYS, quarter * 32 + lane, lane_base + (half ? S::V_COL : S::K_COL));
      tmem_store_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(kv_tmem);
    }
    const uint32_t s_addr = lane_base + S::S_COL + half * 32, dp_addr = lane_base + S::DP_COL + half * 32;
    const uint32_t p_addr = lane_base + S::P_COL + half * 16, ds_addr = lane_base + S::DS_COL + half * 16;
    for (int i = u; i < nq && ok; i += 2) {
      uint32_t sr[32], pr[32], po[16], so[16];
      // the statistics of this step have landed with its rows; waiting on their barrier makes them visible here
      ok = warp_wait(q_full(i % S::STAGES), (uint32_t)(i / S::STAGES) & 1u, a.status, SB_TIMEOUT_SMEM_FULL) &&
           warp_wait(s_full(u), (uint32_t)(i >> 1) & 1u, a.status, SB_TIMEOUT_TMEM_FULL);
      if (!ok) break;
      tc_fence_after();
      tmem_load32(s_addr, sr);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_read);
      ok = warp_wait(dp_full(u), (uint32_t)(i >> 1) & 1u, a.status, SB_TIMEOUT_TMEM_FULL);
      if (!ok) break;
      tc_fence_after();
      tmem_load32(dp_addr, pr);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(dp_read);
      if (a.Tk <= 0) break;                                 // never: a branch keeps the arithmetic below behind the arrivals (see the dq kernel)
      const uint32_t stat = base + S::STAT0 + (i % S::STAGES) * S::STAT;
#pragma unroll
      for (int k = 0; k < 32; k += 4) {
        uint64_t l[2], d[2];
        asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(l[0]), "=l"(l[1]) : "r"(stat + (32 * half + k) * 4));
        asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(d[0]), "=l"(d[1]) : "r"(stat + (BQ + 32 * half + k) * 4));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = k + 2 * e;
          if (Half2<T>::KIND == 0) l[e] = add2(l[e], shift2);
          float x, y;
          split(fma2(pair(sr[j], sr[j + 1]), c2, l[e]), x, y);
          x = ex2(x);
          y = ex2(y);
          uint64_t v = mul2(pair(x, y), add2(pair(pr[j], pr[j + 1]), d[e]));
          if (Half2<T>::KIND == 0) v = mul2(v, f2);
          po[j >> 1] = Half2<T>::pack(x, y);
          split(v, x, y);
          so[j >> 1] = Half2<T>::pack(x, y);
        }
      }
      if (some_hidden && hidden) {
#pragma unroll
        for (int k = 0; k < 16; ++k) po[k] = so[k] = 0u;
      }
      __syncwarp();
      if (i > 0) {                                          // p and ds of the step before have been multiplied
        ok = warp_wait(p_read(u ^ 1), (uint32_t)((i - 1) >> 1) & 1u, a.status, SB_TIMEOUT_TMEM_FULL);
        if (!ok) break;
        tc_fence_after();
      }
      tmem_store16(p_addr, po);
      tmem_store16(ds_addr, so);
      tmem_store_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full(u));
    }
    if (nq > 0 && ok) ok = warp_wait(d_full, 0, a.status, SB_TIMEOUT_TMEM_FULL);
    tc_fence_after();
    if (a.mask) asm volatile("bar.sync 1, 544;" ::: "memory");     // with warp 3
    uint32_t one;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(one) : "r"(one_slot) : "memory");
    const float f = !u ? ex2(-p_shift<T>()) : one ? 0.f : Half2<T>::KIND == 0 ? b.scale / dsf : b.scale;
    // dv by two warpgroups, dk by the others, 64 columns each (DP = 64: one of the two)
    if (splits > 1) {
      if (half < DP / 64) keep_part64<DP>(base + u * 128 * DP * 4, quarter * 32 + lane, half * 64, lane_base + (u ? S::DK_COL : 0) + half * 64, nq > 0 && ok,
                                        hidden);
    } else if (half < DP / 64) {
      const long long off = key < a.Tk ? (((long long)m * a.Tk + key) * a.Hk + hk) * a.D : -1;
      store_acc64<T>(base + ((u * 2 + half) * 4 + quarter) * 4096, lane_base + (u ? S::DK_COL : 0) + half * 64, nq > 0 && ok,
                     f, u ? dk : dv, off, half * 64, a.D, lane, hidden);      // its weights' zeros may have met infinite queries
    }
  }
  if (splits > 1) {
    __syncthreads();
    cluster_sync();
    float dsf;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(dsf) : "r"(scale_slot) : "memory");
    uint32_t one;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(one) : "r"(one_slot) : "memory");
    constexpr int CH = DP / 8;
    for (int x = rank * DKV_THREADS + threadIdx.x; x < 2 * 128 * CH; x += splits * DKV_THREADS) {
      const int u = x / (128 * CH), r = x / CH % 128, c8 = x % CH, key = key0 + r;
      if (key >= a.Tk || c8 * 8 >= a.D) continue;
      join_parts8<T, DP>(base + u * 128 * DP * 4, r, c8, splits, u ? (one ? 0.f : b.scale / dsf) : ex2(-p_shift<T>()),
                         (u ? dk : dv) + (((long long)m * a.Tk + key) * a.Hk + hk) * a.D + c8 * 8);
    }
    cluster_sync();                                          // the others may still read this block's part
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

template <typename T, int DP>
int launch(const SbCrossAttention* g, const XAttnArgs& a, BwdArgs b, void* dq, void* dk, void* dv, cudaStream_t stream) {
  CUtensorMap k64, v64, q64, do64;
  int rc = sb_rows_map(&k64, g->k, g->type, a.D, a.Tk, a.Hk, a.M, g->k_st, g->k_sh, g->k_sb, DqSmem<DP>::BN);
  if (!rc) rc = sb_rows_map(&v64, g->v, g->type, a.D, a.Tk, a.Hk, a.M, g->v_st, g->v_sh, g->v_sb, DqSmem<DP>::BN);
  if (!rc) rc = sb_rows_map(&q64, g->q, g->type, a.D, a.Tq, a.H, a.M * a.G, g->q_st, g->q_sh, g->q_sb, DkvSmem<DP>::BQ);
  if (!rc) rc = sb_rows_map(&do64, b.dout, g->type, a.D, a.Tq, a.H, a.M * a.G, (long long)a.H * a.D, a.D, (long long)a.Tq * a.H * a.D, DkvSmem<DP>::BQ);
  if (!rc) rc = sb_allow_smem((const void*)xattn_dq_kernel<T, DP>, DqSmem<DP>::BYTES);
  if (!rc) rc = sb_allow_smem((const void*)xattn_dkv_kernel<T, DP>, DkvSmem<DP>::BYTES);
  if (rc) return rc;
  b.tiles = (a.R + 127) / 128;
  const long long units = (long long)a.M * a.Hk, gq = units * b.tiles, gk = units * ((a.Tk + 127) / 128);
  if (gq > 0x7ffffffll || gk > 0x7ffffffll) return SB_BAD_ARGUMENT;
  if (Half2<T>::KIND == 0) {
    b.norms = b.peak + gq;
    const int parts = norm_parts(a.Tk);                      // units * parts <= 2 gk is within a grid's limit
    xattn_norms_kernel<DP><<<(unsigned)(units * parts), 256, 0, stream>>>(a, (const __half*)g->v, g->v_sb, g->v_st, g->v_sh, b.norms, parts);
    rc = (int)cudaGetLastError();
    if (rc) return rc;
  }
  using DQ = DqSmem<DP>;
  using DKV = DkvSmem<DP>;
  SbTilePlan plan = {gq, 1};                                 // without dq only the statistics are laid out, by a block per tile
  if (dq) plan = sb_plan_tiles((const void*)xattn_dq_kernel<T, DP>, DQ_THREADS, DQ::BYTES, gq, (a.Tk + DQ::BN - 1) / DQ::BN, DQ_OWN_BLOCKS, DQ_OWN_BLOCKS / 2);
  rc = sb_run_tiles(plan, gq, DQ_THREADS, DQ::BYTES, stream, xattn_dq_kernel<T, DP>, k64, v64, a, b, (uint16_t*)dq);
  if (rc || !dk) return rc;
  const long long steps = (long long)a.G * a.rep * (b.Tqp / DKV::BQ);
  plan = sb_plan_tiles((const void*)xattn_dkv_kernel<T, DP>, DKV_THREADS, DKV::BYTES, gk, (int)(steps < 0x7fffff00 ? steps : 0x7fffff00), DKV_OWN_STEPS,
                       DKV_OWN_STEPS / 2);
  return sb_run_tiles(plan, gk, DKV_THREADS, DKV::BYTES, stream, xattn_dkv_kernel<T, DP>, k64, v64, q64, do64, a, b, (uint16_t*)dk, (uint16_t*)dv);
}

}  // namespace

// out, rest, dout: contiguous [B, Tq, H, D]; out, rest, lse: the forward pass's; ws: 2 * B * H * (Tq rounded up to 64) floats, one per 128 packed
// rows and, in fp16, one per 64 keys of every (memory, key head); dq [B, Tq, H, D] or null; dk, dv
// [M, Tk, Hk, D], both or neither.
SB_API int sb_cross_attention_bwd(const SbCrossAttention* g, const void* out, const void* rest, const void* dout, const float* lse, float* ws, void* dq,
                                  void* dk, void* dv, cudaStream_t stream) {
  XAttnArgs a;
  const int rc = sb_xattn_args(g, &a);
  if (rc) return rc;
  if (!out || !rest || !dout || !lse || !ws || (dk != nullptr) != (dv != nullptr) || (((uintptr_t)dout | (uintptr_t)ws) & 15)) return SB_BAD_ARGUMENT;
  BwdArgs b = {};
  b.dout = (const uint16_t*)dout;
  b.out = (const uint16_t*)out;
  b.rest = (const uint16_t*)rest;
  b.lse = lse;
  b.Tqp = (a.Tq + 63) / 64 * 64;
  b.nlse = ws;
  b.ndelta = ws + (long long)a.M * a.G * a.H * b.Tqp;
  b.peak = b.ndelta + (long long)a.M * a.G * a.H * b.Tqp;
  b.scale = g->scale;
  if (g->type == 0)
    return a.D <= 64 ? launch<__nv_bfloat16, 64>(g, a, b, dq, dk, dv, stream) : launch<__nv_bfloat16, 128>(g, a, b, dq, dk, dv, stream);
  return a.D <= 64 ? launch<__half, 64>(g, a, b, dq, dk, dv, stream) : launch<__half, 128>(g, a, b, dq, dk, dv, stream);
}
