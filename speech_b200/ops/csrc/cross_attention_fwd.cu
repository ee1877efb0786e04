// Fused cross attention, forward, for many query rows:  o = softmax(scale q k^T) v  without the score matrix in memory.
//
// One pass over the keys with the running maximum m and sum l of every row; p = 2^(c s - c m) is held unnormalised:
//   s = q k_j^T,  m' = max(m, max s),  o = o 2^(c (m - m')) + p v_j,  l = l 2^(c (m - m')) + sum p,  at the end o / w
// with w the sum of p as it is rounded for the product with v (below), and lse = c m + log2 l is kept for the backward pass (+inf for a row
// that sees nothing: its probabilities are then 2^-inf = 0).
//
// A CTA takes two tiles of 128 packed rows and streams blocks of 64 keys of its memory and key head past both, so that keys and values
// cross the L2 once per 256 rows.  Warp 0 loads keys and values by TMA, warps 1 and 3 issue the tcgen05.mma of a tile each, warp 2
// clears the rows of hidden keys and lays out their addends (one more step of the score product), and one warpgroup per row tile does the
// softmax: scores and output accumulate in tensor memory (per tile two buffers of 64 columns and DP columns), the probabilities go back
// there as 16-bit pairs over the scores they came from and are the A operand of the second product.  The scores of the next block are there before the softmax of this
// one ends; with one buffer of 128 keys the warpgroups waited for the tensor core and it for them (41 % of its cycles busy).  The output is rescaled only when a row's maximum
// has grown by more than 2^8 since the last time; p then stays below 2^8, and the result does not depend on it beyond rounding.
// Where there are fewer tile pairs than SMs, up to eight CTAs of a cluster share one, each with its part of the keys; unnormalised outputs
// and (m, w, l) meet in shared memory and are joined in a fixed order: f_i = 2^(c (m_i - max m)), o = sum f_i o_i / sum f_i w_i.
//
// Rounding: scores, maxima, sums and output are fp32; p is rounded to the operands' 16-bit type, which is what the tensor core
// multiplies (up to 2^-8 of a weight in bf16), and the output is divided by the sum w of the rounded weights.  Divided by l it would be off by the
// rounding of the largest weight where one key leads (a weight up to 2^8, because of the maximum that stands still): a common factor, which the
// backward pass's delta = sum do o takes on and subtracts from values of its own size.  [Rows that one of 512 keys leads by 3 / 4 / 5 nats, bf16: dq
// off by 11 / 17 / 60 % of its norm; so by 1 %.]  lse is the unrounded p's.
#include "cross_attention.cuh"
#include "cross_attention_host.h"

namespace {

constexpr int FWD_THREADS = 384;
constexpr int BN = 64;
// What a CTA takes besides its blocks, and what a join takes, in blocks.  [1 x 100 queries, 8 heads of 128, 1 / 2 / 4 / 8 CTAs a tile:
// 102 / 63 / 43 / 33 us for 7500 keys, 33 / 29 / 25 / 25 for 1500, 20 / 23 / 23 / 21 for 500]
constexpr int OWN_BLOCKS = 9;
template <int DP> struct FwdSmem {
  static constexpr int STAGES = 4;
  static constexpr int TILE = 128 * DP * 2, KEYS = BN * DP * 2;      // 128 query rows, a block of keys or values
  static constexpr int K0 = 2 * TILE, V0 = K0 + STAGES * KEYS, BAR = V0 + STAGES * KEYS;
  static constexpr int ONES0 = BAR + 512, ADD0 = ONES0 + ONES_BYTES, BYTES = ADD0 + STAGES * ADDEND_BYTES + 1024;
};

// KEEP: rest and lse are written for a backward pass.
template <typename T, int DP, bool KEEP>
__global__ void __launch_bounds__(FWD_THREADS, 1)
xattn_fwd_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const XAttnArgs a, uint16_t* __restrict__ out,
                 uint16_t* __restrict__ rest, float* __restrict__ lse, const long long tile0, const int splits) {
  using S = FwdSmem<DP>;
  constexpr int HALVES = DP / 64;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bars = base + S::BAR;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto k_full = [&](int s) { return bars + 8u * s; };
  auto k_empty = [&](int s) { return bars + 8u * (4 + s); };
  auto k_clean = [&](int s) { return bars + 8u * (34 + s); };
  auto v_full = [&](int s) { return bars + 8u * (8 + s); };
  auto v_clean = [&](int s) { return bars + 8u * (12 + s); };
  auto v_empty = [&](int s) { return bars + 8u * (16 + s); };
  auto s_full = [&](int t, int u) { return bars + 8u * (20 + 2 * t + u); };
  auto p_full = [&](int t, int u) { return bars + 8u * (24 + 2 * t + u); };
  auto pv_done = [&](int t) { return bars + 8u * (28 + t); };   // every block's product: at most one is outstanding when it is waited for
  auto o_full = [&](int t) { return bars + 8u * (32 + t); };    // the last one
  const uint32_t q_ready = bars + 8u * 30, tmem_slot = bars + 8u * 31, seen_slot = bars + 8u * 40;      // seen: whether the mask leaves any of these keys

  const int pairs = (a.R + 255) / 256;                    // row-tile pairs of a (memory, key head): neighbours in the grid, for the L2
  const int local = blockIdx.x / splits, rank = blockIdx.x - local * splits;      // block `rank` of a cluster takes its part of the keys
  const int index = (int)tile0 + local;
  const int unit = index / pairs, m = unit / a.Hk, hk = unit % a.Hk;
  const int row0 = (index - unit * pairs) * 256;
  const int tiles = a.R - row0 > 128 ? 2 : 1;
  const int len = visible_keys(a, m);
  const int blocks = (len + BN - 1) / BN, share = (blocks + splits - 1) / splits, first = rank * share * BN;
  const int nt = min(share, max(0, blocks - rank * share));
  const bool hide = a.mask != nullptr;

  init_addends<T>(base + S::ONES0, S::STAGES, threadIdx.x, FWD_THREADS);
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      // empty: the tiles' products and the warp that clears.  That warp looks at every block, also where no product waits for it; were it not
      // counted, a stage could be filled twice under it, and the parity of its next wait, and of a wait for it, would be another phase's.
      mbar_init(k_full(s), 1); mbar_init(k_clean(s), 1); mbar_init(k_empty(s), tiles + 1);
      mbar_init(v_full(s), 1); mbar_init(v_clean(s), 1); mbar_init(v_empty(s), tiles + 1);
    }
    for (int t = 0; t < 2; ++t) {
      for (int u = 0; u < 2; ++u) { mbar_init(s_full(t, u), 1); mbar_init(p_full(t, u), 4); }
      mbar_init(pv_done(t), 1);
      mbar_init(o_full(t), 1);
    }
    mbar_init(q_ready, 4 * tiles);
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
    // ---------------------------------------------------------------- loads
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    int issued = 0;
    for (int j = 0; j < nt && ok; ++j) {
      ok = warp_wait(k_empty(s), ph ^ 1u, a.status, SB_TIMEOUT_SMEM_EMPTY);
      if (!ok) break;
      if (elect_one()) {
        mbar_expect_tx(k_full(s), S::KEYS);
#pragma unroll
        for (int h = 0; h < HALVES; ++h) tma_load_4d(base + S::K0 + s * S::KEYS + h * (BN * 128), &map_k, k_full(s), h * 64, first + j * BN, hk, m);
      }
      __syncwarp();
      ok = warp_wait(v_empty(s), ph ^ 1u, a.status, SB_TIMEOUT_SMEM_EMPTY);
      issued = j + 1;
      if (!ok) break;
      if (elect_one()) {
        mbar_expect_tx(v_full(s), S::KEYS);
#pragma unroll
        for (int h = 0; h < HALVES; ++h) tma_load_4d(base + S::V0 + s * S::KEYS + h * (BN * 128), &map_v, v_full(s), h * 64, first + j * BN, hk, m);
      }
      __syncwarp();
      if (++s == S::STAGES) { s = 0; ph ^= 1u; }
    }
    // no copy may be in flight when the block ends: the last one of every stage has landed (long since, unless a wait gave up)
    for (int i = issued > S::STAGES ? issued - S::STAGES : 0; i < issued; ++i) {
      warp_wait(k_full(i % S::STAGES), (uint32_t)(i / S::STAGES) & 1u, a.status, SB_TIMEOUT_SMEM_FULL);
      if (ok || i + 1 < issued) warp_wait(v_full(i % S::STAGES), (uint32_t)(i / S::STAGES) & 1u, a.status, SB_TIMEOUT_SMEM_FULL);
    }
  } else if (warp == 1 || (warp == 3 && tiles == 2)) {
    // ---------------------------------------------------------------- matrix products of one row tile
    const int t = warp >> 1;
    constexpr uint32_t idesc_s = instr_desc<T>(BN, false), idesc_o = instr_desc<T>(DP, true);
    const uint64_t qd = make_desc(base + t * S::TILE, 16, 1024), kd = make_desc(base + S::K0, 16, 1024), vd = make_desc(base + S::V0, BN * 128, 1024);
    auto scores = [&](int j) {                              // s = q k^T of block j into buffer j & 1
      const uint64_t st = (uint64_t)(((j % S::STAGES) * S::KEYS) >> 4);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint64_t ro = (uint64_t)(((kk >> 2) * 16384 + (kk & 3) * 32) >> 4), ko = (uint64_t)(((kk >> 2) * (BN * 128) + (kk & 3) * 32) >> 4);
          umma_bf16(tmem + t * 128 + (j & 1) * 64, qd + ro, kd + st + ko, idesc_s, kk > 0);
        }
        if (hide || first + (j + 1) * BN > len)
          umma_bf16(tmem + t * 128 + (j & 1) * 64, make_desc_plain(base + S::ONES0), make_desc_plain(base + S::ADD0 + (j % S::STAGES) * ADDEND_BYTES), idesc_s, 1);
        umma_commit(s_full(t, j & 1));
        umma_commit(k_empty(j % S::STAGES));
      }
      __syncwarp();
    };
    // A block has landed, and where it has hidden keys they have been cleared: in this order, because only a block that has landed says that the
    // clearing of its stage's last one is done.
    auto landed = [&](int j, uint32_t full, uint32_t clean) {
      const uint32_t ph = (uint32_t)(j / S::STAGES) & 1u;
      return warp_wait(full, ph, a.status, SB_TIMEOUT_SMEM_FULL) &&
             (!(hide || first + (j + 1) * BN > len) || warp_wait(clean, ph, a.status, SB_TIMEOUT_SMEM_FULL));
    };
    bool ok = nt > 0 && warp_wait(q_ready, 0, a.status, SB_TIMEOUT_SMEM_FULL);
    for (int j = 0; j < 2 && j < nt && ok; ++j) {
      ok = landed(j, k_full(j), k_clean(j));
      if (!ok) break;
      tc_fence_after();
      scores(j);
    }
    for (int j = 0; j < nt && ok; ++j) {
      const int s = j % S::STAGES;
      ok = landed(j, v_full(s), v_clean(s)) && warp_wait(p_full(t, j & 1), (uint32_t)(j >> 1) & 1u, a.status, SB_TIMEOUT_TMEM_EMPTY);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk)
          umma_ts(tmem + 256 + t * DP, tmem + t * 128 + (j & 1) * 64 + kk * 8, vd + (uint64_t)((s * S::KEYS + kk * 2048) >> 4), idesc_o, (j > 0) | (kk > 0));
        umma_commit(v_empty(s));
        umma_commit(j == nt - 1 ? o_full(t) : pv_done(t));
      }
      __syncwarp();
      if (j + 2 < nt) {
        const int s2 = (j + 2) % S::STAGES;
        ok = landed(j + 2, k_full(s2), k_clean(s2));
        if (!ok) break;
        tc_fence_after();
        scores(j + 2);
      }
    }
  } else if (warp == 2) {
    // ---------------------------------------------------------------- hidden keys: their rows cleared, their scores' addends
    int s = 0;
    uint32_t ph = 0;
    bool hid[2] = {hidden_key(a, m, len, first + lane), hidden_key(a, m, len, first + 32 + lane)};      // this lane's keys of block j, read a block ahead
    bool seen = false;
    for (int j = 0; j < nt; ++j) {
      const bool some = hide || first + (j + 1) * BN > len;
      uint32_t w[2] = {0, 0};
      if (some) {
#pragma unroll
        for (int i = 0; i < 2; ++i) w[i] = __ballot_sync(0xffffffffu, hid[i]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) hid[i] = hidden_key(a, m, len, first + (j + 1) * BN + 32 * i + lane);
      if (!warp_wait(k_full(s), ph, a.status, SB_TIMEOUT_SMEM_FULL)) break;
      if (some) {
        clear_rows<DP>(base + S::K0 + s * S::KEYS, w, lane);
        store_addends<T>(base + S::ADD0 + s * ADDEND_BYTES, w, lane);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(k_clean(s));
        mbar_arrive(k_empty(s));
      }
      if (!warp_wait(v_full(s), ph, a.status, SB_TIMEOUT_SMEM_FULL)) break;
      if (some) {
        clear_rows<DP>(base + S::V0 + s * S::KEYS, w, lane);
        seen |= (w[0] & w[1]) != 0xffffffffu;
        if (j == nt - 1 && lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(seen_slot), "r"((uint32_t)seen) : "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(v_clean(s));
        mbar_arrive(v_empty(s));
      }
      if (++s == S::STAGES) { s = 0; ph ^= 1u; }
    }
  } else if (warp >= 4 && (warp - 4) / 4 < tiles) {
    // ---------------------------------------------------------------- softmax and output of one row tile
    const int t = (warp - 4) >> 2, quarter = warp & 3;
    const int tile_row = row0 + t * 128, row = tile_row + quarter * 32 + lane;
    bool ok = true;
    float mx = -INFINITY, l = 0.f, w = 0.f;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t o_addr = lane_base + 256 + t * DP;
    if (nt > 0) {
      load_rows<DP>(a.q, row_offset(a, a.q_sb, a.q_st, a.q_sh, m, hk, row), a.D, base + t * S::TILE, quarter, lane);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
    }
    for (int j = 0; j < nt; ++j) {
      const uint32_t s_addr = lane_base + t * 128 + (j & 1) * 64;
      ok = warp_wait(s_full(t, j & 1), (uint32_t)(j >> 1) & 1u, a.status, SB_TIMEOUT_TMEM_FULL);
      if (!ok) break;
      tc_fence_after();
      uint32_t r[BN];
      tmem_load64(s_addr, r);
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int k = 0; k < BN; k += 8)
#pragma unroll
        for (int i = 0; i < 4; ++i) top[i] = max3(top[i], __uint_as_float(r[k + 2 * i]), __uint_as_float(r[k + 2 * i + 1]));
      const float tile_max = fmaxf(max3(top[0], top[1], top[2]), top[3]);
      // the output keeps its scale until a row's maximum has grown by 2^8
      const bool grow = mx == -INFINITY ? false : (tile_max - mx) * a.c > 8.f;
      if (__any_sync(0xffffffffu, grow)) {
        const float nm = fmaxf(mx, tile_max);
        const float f = mx == -INFINITY ? 1.f : ex2((mx - nm) * a.c);
        if (mx != -INFINITY) {
          l *= f;
          w *= f;
          mx = nm;
        }
        if (j > 0) {
          // products up to block j - 1 have been added: those up to j - 2 have (the scores of block j were issued behind them), and the
          // last one is waited for here
          ok = warp_wait(pv_done(t), (uint32_t)(j - 1) & 1u, a.status, SB_TIMEOUT_TMEM_FULL);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < DP / 32; ++i) {
            uint32_t x[32];
            tmem_load32(o_addr + 32 * i, x);
#pragma unroll
            for (int k = 0; k < 32; ++k) x[k] = __float_as_uint(__uint_as_float(x[k]) * f);
            tmem_store32(o_addr + 32 * i, x);
          }
        }
      }
      if (mx == -INFINITY) mx = tile_max;                  // nothing seen so far: output and sum are zero at any scale
      const float mc = mx == -INFINITY ? 0.f : mx * a.c;
      const uint64_t c2 = pair(a.c, a.c), shift2 = pair(-mc, -mc);
      uint64_t sum[2] = {0, 0}, rounded[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < BN / 32; ++i) {
        uint32_t p[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          float x, y;
          split(fma2(pair(r[32 * i + 2 * k], r[32 * i + 2 * k + 1]), c2, shift2), x, y);
          x = ex2(x);
          y = ex2(y);
          if (KEEP) sum[k & 1] = add2(sum[k & 1], pair(x, y));
          p[k] = Half2<T>::pack(x, y);
          const float2 back = Half2<T>::unpack(p[k]);
          rounded[k & 1] = add2(rounded[k & 1], pair(back.x, back.y));
        }
        tmem_store16(s_addr + 16 * i, p);
      }
      {
        float x, y;
        split(add2(sum[0], sum[1]), x, y);
        l += x + y;
        split(add2(rounded[0], rounded[1]), x, y);
        w += x + y;
      }
      tmem_store_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full(t, j & 1));
    }
    if (nt > 0 && ok) ok = warp_wait(o_full(t), 0, a.status, SB_TIMEOUT_TMEM_FULL);
    tc_fence_after();
    if (hide && nt > 0 && ok) {
      // a mask that leaves nothing: the output is zero whatever the query holds (its infinities met the cleared keys' zeros)
      uint32_t seen = 1;
      ok = warp_wait(v_clean((nt - 1) % S::STAGES), (uint32_t)((nt - 1) / S::STAGES) & 1u, a.status, SB_TIMEOUT_SMEM_FULL);
      if (ok) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(seen) : "r"(seen_slot) : "memory");
      if (!seen) {
        mx = -INFINITY;
        l = w = 0.f;
        ok = false;
      }
    }
    if (splits > 1) {
      asm volatile("bar.sync 2, %0;" ::"r"(tiles * 128) : "memory");     // no product of either tile reads shared memory any more
      const int r = t * 128 + quarter * 32 + lane;
#pragma unroll
      for (int i = 0; i < DP / 64; ++i) keep_part64<DP>(base, r, 64 * i, o_addr + 64 * i, nt > 0 && ok);
      asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(base + 256 * DP * 4 + r * 8), "f"(mx), "f"(w) : "memory");
      if (KEEP) asm volatile("st.shared.f32 [%0], %1;" ::"r"(base + 256 * (DP * 4 + 8) + r * 4), "f"(l) : "memory");
    } else {
      const long long at_row = row_offset(a, (long long)a.Tq * a.H * a.D, (long long)a.H * a.D, a.D, m, hk, row);
      if (KEEP && row < a.R) lse[(long long)unit * a.R + row] = l > 0.f ? fmaf(mx, a.c, log2f(l)) : (l == 0.f ? INFINITY : l);
      __syncwarp();                                          // whole warps again for the loads below
      const float inv = w == 0.f ? 0.f : 1.f / w;
      const uint32_t buf = base + t * S::TILE + quarter * 4096;      // the tile's queries have been read
#pragma unroll
      for (int i = 0; i < DP / 64; ++i) {
        uint32_t r[64], v[32], off[32];
        if (nt > 0 && ok) {
          tmem_load64(o_addr + 64 * i, r);
        } else {
#pragma unroll
          for (int k = 0; k < 64; ++k) r[k] = 0u;
        }
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = out_pair<T>(__uint_as_float(r[2 * k]) * inv, __uint_as_float(r[2 * k + 1]) * inv, off[k]);
        store_rows64(buf, v, out, at_row, 64 * i, a.D, lane);
        if (KEEP) store_rows64(buf, off, rest, at_row, 64 * i, a.D, lane);
      }
    }
  }
  if (splits > 1) {
    __syncthreads();
    cluster_sync();
    constexpr int CH = DP / 8;
    for (int x = rank * FWD_THREADS + threadIdx.x; x < tiles * 128 * CH; x += splits * FWD_THREADS) {
      const int r = x / CH, c8 = x % CH, row = row0 + r;
      if (row >= a.R || c8 * 8 >= a.D) continue;
      const uint32_t ml = base + 256 * DP * 4 + r * 8;
      float top = -INFINITY, sum = 0.f, l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int i = 0; i < splits; ++i) top = fmaxf(top, load_remote2(in_block(ml, i)).x);
      for (int i = 0; i < splits; ++i) {
        const float2 v = load_remote2(in_block(ml, i));
        if (v.y == 0.f) continue;                            // saw nothing
        const float f = ex2((v.x - top) * a.c);
        sum = fmaf(f, v.y, sum);
        if (KEEP && c8 == 0) l = fmaf(f, load_remote(in_block(base + 256 * (DP * 4 + 8) + r * 4, i)), l);
        add_part8<DP>(base, r, c8, i, f, o);
      }
      if (KEEP && c8 == 0) lse[(long long)unit * a.R + row] = l > 0.f ? fmaf(top, a.c, log2f(l)) : (l == 0.f ? INFINITY : l);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const long long at = row_offset(a, (long long)a.Tq * a.H * a.D, (long long)a.H * a.D, a.D, m, hk, row) + c8 * 8;
      uint32_t v[4], off[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = out_pair<T>(o[2 * k] * inv, o[2 * k + 1] * inv, off[k]);
      *reinterpret_cast<uint4*>(out + at) = make_uint4(v[0], v[1], v[2], v[3]);
      if (KEEP) *reinterpret_cast<uint4*>(rest + at) = make_uint4(off[0], off[1], off[2], off[3]);
    }
    cluster_sync();                                          // the others may still read this block's part
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

template <typename T, int DP, bool KEEP>
int launch(const XAttnArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, void* out, void* rest, float* lse, cudaStream_t stream) {
  const long long grid = (long long)((a.R + 255) / 256) * a.M * a.Hk;
  if (grid > 0x7ffffffll) return SB_BAD_ARGUMENT;
  const auto kernel = xattn_fwd_kernel<T, DP, KEEP>;
  const int rc = sb_allow_smem((const void*)kernel, FwdSmem<DP>::BYTES);
  if (rc) return rc;
  const SbTilePlan plan = sb_plan_tiles((const void*)kernel, FWD_THREADS, FwdSmem<DP>::BYTES, grid, (a.Tk + BN - 1) / BN, OWN_BLOCKS, OWN_BLOCKS);
  return sb_run_tiles(plan, grid, FWD_THREADS, FwdSmem<DP>::BYTES, stream, kernel, mk, mv, a, (uint16_t*)out, (uint16_t*)rest, lse);
}
template <typename T>
int launch(const XAttnArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, void* out, void* rest, float* lse, cudaStream_t stream) {
  if (a.D <= 64) return lse ? launch<T, 64, true>(a, mk, mv, out, rest, lse, stream) : launch<T, 64, false>(a, mk, mv, out, rest, lse, stream);
  return lse ? launch<T, 128, true>(a, mk, mv, out, rest, lse, stream) : launch<T, 128, false>(a, mk, mv, out, rest, lse, stream);
}

}  // namespace

// q [B, Tq, H, D], k / v [M, Tk, Hk, D] by element strides (batch, time, head); out contiguous [B, Tq, H, D]; for a backward pass
// rest [B, Tq, H, D], what rounding took from out, and lse fp32 [M, Hk, R], else both null; ws: sb_cross_attention_workspace() bytes.
SB_API int sb_cross_attention_fwd(const SbCrossAttention* g, void* out, void* rest, float* lse, void* ws, cudaStream_t stream) {
  XAttnArgs a;
  int rc = sb_xattn_args(g, &a);
  if (rc) return rc;
  if (!out || (rest != nullptr) != (lse != nullptr)) return SB_BAD_ARGUMENT;
  if (sb_few_rows(g)) return sb_step_cross_attention(g, out, rest, lse, ws, stream);
  CUtensorMap mk, mv;
  rc = sb_rows_map(&mk, g->k, g->type, a.D, a.Tk, a.Hk, a.M, g->k_st, g->k_sh, g->k_sb, BN);
  if (!rc) rc = sb_rows_map(&mv, g->v, g->type, a.D, a.Tk, a.Hk, a.M, g->v_st, g->v_sh, g->v_sb, BN);
  if (rc) return rc;
  return g->type == 0 ? launch<__nv_bfloat16>(a, mk, mv, out, rest, lse, stream) : launch<__half>(a, mk, mv, out, rest, lse, stream);
}
