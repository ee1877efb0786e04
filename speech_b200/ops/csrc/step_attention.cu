// Attention for a few query rows per key head: one decoding step over an encoder's states, or over a prompt that a group of rows
// shares together with every row's own cache; also the forward pass of short queries in training.
//
// Keys and values are read once and little is computed on them, so bytes bound it, and what counts is how many loads are in flight.
// The keys of a (memory, key head) are split over blocks and over the four warps of a block; every warp streams tiles of 16 keys through
// a ring of its own in shared memory (cp.async, 16 or 24 KB per warp, 190 KB per SM; no barrier between warps), takes
// its fragments of mma.m16n8k16 from there with ldmatrix, and keeps running maximum m, sum l (of rounded weights: w) and the unnormalised output in
// registers.
// The parts are joined in the block; up to eight blocks of a (memory, key head) are a cluster and join theirs through one another's
// shared memory, more blocks, and the two kinds of keys of a shared prompt, through memory and a second small kernel:
//   o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) w_i.
// Loads straight into registers (16 keys ahead, 228 registers, or fewer and spills) reached a third of this.
//
// Packed rows (rows that read the same keys: group x heads of a key head x tokens, as in cross_attention.cuh) fill blocks of 16, one or
// two per warp; more rows than 32 read the keys again, from the L2.
//
// Rounding: as in cross_attention_fwd.cu (weights rounded to 16 bits for the second product and for the sum that divides it, all else fp32).
#include "cross_attention_host.h"

namespace {

struct Segment {
  const uint16_t *k, *v;
  long long k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  const int* lengths;       // [memories] or null
  const uint8_t* mask;      // [memories, size] or null
  int size;                 // positions
  int rows_per;             // batch rows of a memory (G; 1 for own caches)
  int causal;               // token t sees its row's first length - Tq + 1 + t positions
  int R;                    // packed rows of a (memory, key head)
  int row_groups;           // blocks over the rows
  int splits, chunk;        // blocks over the keys, keys of one
  int blocks;
};

struct StepArgs {
  const uint16_t* q;
  long long q_sb, q_st, q_sh;
  int B, Tq, H, Hk, rep, D;
  float c;
  Segment seg[2];
  int slots;                // splits of both segments
  int cluster;              // the splits of a unit are a cluster: no partial results in memory
  uint16_t *out, *rest;     // [B, Tq, H, D]; rest: what rounding took from out, or null
  float* lse;               // packed rows of segment 0, or null
  float* part_o;            // [slots, B * Tq * H, D]
  float2* part_mw;          // [slots, B * Tq * H]: maximum, sum of rounded weights
  float* part_l;            // the same: sum of the weights, where lse is wanted
};

template <typename T> __device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__half>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16 bytes from global to shared memory, or 16 zero bytes
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
// 16-byte chunk `ch` of row `row` in a tile of rows of DP 16-bit elements; the XOR spreads the eight rows of an ldmatrix over all banks
template <int DP> __device__ __forceinline__ uint32_t row_addr(uint32_t base, int row, int ch) {
  return base + (uint32_t)(row * DP * 2) + (uint32_t)((ch ^ (row & 7)) << 4);
}

constexpr int STEP_THREADS = 128;
template <int DP, int MT> struct StepSmem {
  static constexpr int HALF = 16 * DP * 2;                 // 16 rows of keys or values
  static constexpr int RING = (DP == 128 ? 1 : 2) * (MT == 1 ? 2 : 3);      // tiles of keys and values per warp
  static constexpr int Q0 = 4 * RING * 2 * HALF, BYTES = Q0 + MT * HALF + 16;
  static constexpr int BLOCKS = MT == 1 ? 3 : 2;           // per SM
};

// packed row r of (mem, hk) as a row of the [B, Tq, H] output
__device__ __forceinline__ long long query_row(const StepArgs& a, const Segment& s, int mem, int hk, int r) {
  const int y = r / a.Tq, t = r - y * a.Tq, gr = y / a.rep;
  return ((long long)(mem * s.rows_per + gr) * a.Tq + t) * a.H + hk * a.rep + y - gr * a.rep;
}
template <typename T>
__device__ __forceinline__ void write_row(const StepArgs& a, const Segment& s, int mem, int hk, int r, int d, float big, float l, float w, const float* v) {
  const long long qrow = query_row(a, s, mem, hk, r);
  const float inv = w == 0.f ? 0.f : 1.f / w;
  uint32_t o4[4], r4[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) o4[k] = out_pair<T>(v[2 * k] * inv, v[2 * k + 1] * inv, r4[k]);
  *reinterpret_cast<uint4*>(a.out + qrow * a.D + d) = make_uint4(o4[0], o4[1], o4[2], o4[3]);
  if (a.rest) *reinterpret_cast<uint4*>(a.rest + qrow * a.D + d) = make_uint4(r4[0], r4[1], r4[2], r4[3]);
  if (a.lse && d == 0) a.lse[((long long)mem * a.Hk + hk) * s.R + r] = l > 0.f ? big + log2f(l) : (l == 0.f ? INFINITY : l);
}
// two floats at a shared-memory address of block `rank` of the cluster
__device__ __forceinline__ float2 remote_float2(uint32_t addr, int rank) { return load_remote2(in_block(addr, rank)); }

// MT: row blocks of 16 per warp; KEEP: lse is written for a backward pass, which takes the sum of the unrounded weights too
template <typename T, int DP, int MT, bool KEEP>
__global__ void __launch_bounds__(STEP_THREADS, (StepSmem<DP, MT>::BLOCKS)) step_kernel(const __grid_constant__ StepArgs a) {
  using S = StepSmem<DP, MT>;
  constexpr int CH = DP / 8, NT = DP / 8, KS = DP / 16;
  __shared__ float s_m[4][16 * MT], s_l[4][16 * MT], s_w[4][16 * MT], s_join_l[16 * MT];
  __shared__ float2 s_join[16 * MT];
  extern __shared__ __align__(16) uint8_t smem_raw[];
  const uint32_t base = smem_u32(smem_raw), qs = base + S::Q0;
  const int second = blockIdx.x >= a.seg[0].blocks ? 1 : 0;
  const Segment& s = a.seg[second];
  int x = blockIdx.x - (second ? a.seg[0].blocks : 0);
  const int split = x % s.splits;
  x /= s.splits;
  const int rg = x % s.row_groups;
  x /= s.row_groups;
  const int hk = x % a.Hk, mem = x / a.Hk;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int row0 = rg * 16 * MT;

  int len = s.size;
  if (s.lengths) len = min(max(s.lengths[mem], 0), s.size);
  const int key_begin = split * s.chunk, key_end = min(len, key_begin + s.chunk);
  const int tiles = key_end > key_begin ? (key_end - key_begin + 15) / 16 : 0;
  const uint8_t* mask = s.mask ? s.mask + (long long)mem * s.size : nullptr;

  // ---- the ring: tile i of the block belongs to warp i % 4
  const int sub = lane / CH, ch = lane % CH;               // 32 / CH rows per instruction
  const bool on = ch * 8 < a.D;                            // chunks behind the head size are zeros
  const uint16_t* kp = s.k + (long long)mem * s.k_sb + (long long)hk * s.k_sh;
  const uint16_t* vp = s.v + (long long)mem * s.v_sb + (long long)hk * s.v_sh;
  const uint16_t *k_at = kp, *v_at = vp;                   // this lane's first chunk of tile `next`
  if (on) {
    k_at += (long long)(key_begin + warp * 16 + sub) * s.k_st + ch * 8;
    v_at += (long long)(key_begin + warp * 16 + sub) * s.v_st + ch * 8;
  }
  const long long k_step = on ? s.k_st * (32 / CH) : 0, v_step = on ? s.v_st * (32 / CH) : 0;
  const uint32_t ring = base + warp * (S::RING * 2 * S::HALF);
  const uint32_t lane_at = (uint32_t)(sub * DP * 2);
  auto fetch = [&](int i, int slot) {                      // one commit group per call, empty behind the last tile
    if (i < tiles) {
      const int left = key_end - (key_begin + i * 16);     // keys from this tile on
      const uint32_t kt = ring + slot * (2 * S::HALF) + lane_at, vt = kt + S::HALF;
      const uint16_t *kq = k_at, *vq = v_at;
      if (left >= 16 && !mask) {
#pragma unroll
        for (int r = 0; r < 16; r += 32 / CH) {
          const uint32_t x = (uint32_t)(r * DP * 2) + (uint32_t)((ch ^ ((r + sub) & 7)) << 4);
          copy16(kt + x, kq, on);
          copy16(vt + x, vq, on);
          kq += k_step;
          vq += v_step;
        }
      } else {
#pragma unroll 1
        for (int r = 0; r < 16; r += 32 / CH) {
          const uint32_t x = (uint32_t)(r * DP * 2) + (uint32_t)((ch ^ ((r + sub) & 7)) << 4);
          const bool in = on && r + sub < left;
          const bool see = in && !(mask && mask[key_begin + i * 16 + r + sub]);      // a hidden value never meets its zero weight
          copy16(kt + x, in ? kq : kp, in);
          copy16(vt + x, see ? vq : vp, see);
          kq += k_step;
          vq += v_step;
        }
      }
      k_at += k_step * (2 * CH);                           // 64 rows on
      v_at += v_step * (2 * CH);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int next = warp;
#pragma unroll
  for (int i = 0; i < S::RING - 1; ++i, next += 4) fetch(next, i);

  // ---- query rows: packed row -> (batch row, token, head)
  for (int i = threadIdx.x; i < MT * 16 * CH; i += STEP_THREADS) {
    const int lr = i / CH, qc = i % CH, r = row0 + lr;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < s.R && qc * 8 < a.D) {
      const int y = r / a.Tq, t = r - y * a.Tq, gr = y / a.rep;
      v = *reinterpret_cast<const uint4*>(a.q + (long long)(mem * s.rows_per + gr) * a.q_sb + (long long)t * a.q_st +
                                          (long long)(hk * a.rep + y - gr * a.rep) * a.q_sh + qc * 8);
    }
    st_shared_v4(row_addr<DP>(qs, lr, qc), v.x, v.y, v.z, v.w);
  }
  int seen[MT][2];                                         // keys that rows g and g + 8 of each row block see
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = row0 + 16 * t + g + 8 * u;
      seen[t][u] = r >= s.R ? 0 : (s.causal ? len - a.Tq + 1 + r % a.Tq : len);
    }
  __syncthreads();

  const int mrow = (lane & 7) + ((lane >> 3) & 1) * 8, mch = lane >> 4;      // ldmatrix rows of Q and V: (row half, chunk) by lane group
  uint32_t qf[MT == 1 ? KS : 1][4];
  if (MT == 1) {
#pragma unroll
    for (int k = 0; k < KS; ++k) ldmatrix4(row_addr<DP>(qs, mrow, 2 * k + mch), qf[MT == 1 ? k : 0]);
  }
  float m[MT][2], l[MT][2], w[MT][2], o[MT][NT][4];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    m[t][0] = m[t][1] = -INFINITY;
    l[t][0] = l[t][1] = w[t][0] = w[t][1] = 0.f;
#pragma unroll
    for (int i = 0; i < NT; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
  }

  int slot = 0;
  const int all_see = mask ? 0 : min(key_end, s.causal ? len - a.Tq + 1 : len);      // every row sees the keys below
  for (int i = warp; i < tiles; i += 4) {
    {
      int free_slot = slot + S::RING - 1;
      if (free_slot >= S::RING) free_slot -= S::RING;
      __syncwarp();                                        // the whole warp is done with the tile that is overwritten
      fetch(next, free_slot);
      next += 4;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(S::RING - 1) : "memory");
    __syncwarp();
    const uint32_t kt = ring + slot * (2 * S::HALF), vt = kt + S::HALF;
    if (++slot == S::RING) slot = 0;
    const int key0 = key_begin + i * 16;
    float sc[MT][2][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int n = 0; n < 2; ++n) sc[t][n][0] = sc[t][n][1] = sc[t][n][2] = sc[t][n][3] = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      uint32_t kf[4];
      ldmatrix4(row_addr<DP>(kt, (lane & 7) + mch * 8, 2 * k + ((lane >> 3) & 1)), kf);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        uint32_t q2[4];
        if (MT > 1) ldmatrix4(row_addr<DP>(qs, 16 * t + mrow, 2 * k + mch), q2);
        const uint32_t* q = MT == 1 ? qf[MT == 1 ? k : 0] : q2;
        mma16816<T>(sc[t][0], q, kf[0], kf[1]);
        mma16816<T>(sc[t][1], q, kf[2], kf[3]);
      }
    }
    if (key0 + 16 > all_see) {
      // this lane's columns of the scores are keys key0 + {2c, 2c+1, 2c+8, 2c+9}
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = key0 + 2 * c + (e & 1) + 8 * (e >> 1);
        const bool see = key < key_end && !(mask && mask[key]);
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int u = 0; u < 2; ++u)
            if (!(see && key < seen[t][u])) sc[t][e >> 1][2 * u + (e & 1)] = -INFINITY;
      }
    }
    uint32_t p[MT][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) {                        // row g + 8 u: columns sc[.][n][2u], sc[.][n][2u + 1]
        float v[4] = {sc[t][0][2 * u], sc[t][0][2 * u + 1], sc[t][1][2 * u], sc[t][1][2 * u + 1]};
        float mx = fmaxf(max3(v[0], v[1], v[2]), v[3]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) * a.c;
        const bool grow = mx > m[t][u] + 8.f && m[t][u] != -INFINITY;
        if (__any_sync(0xffffffffu, grow)) {               // rare: the output keeps its scale until a maximum has grown by 2^8
          const float nm = m[t][u] == -INFINITY ? m[t][u] : fmaxf(m[t][u], mx);
          const float f = m[t][u] == -INFINITY ? 1.f : ex2(m[t][u] - nm);
          m[t][u] = nm;
          if (KEEP) l[t][u] *= f;
          w[t][u] *= f;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            o[t][n][2 * u] *= f;
            o[t][n][2 * u + 1] *= f;
          }
        }
        if (m[t][u] == -INFINITY) m[t][u] = mx;
        const float from = m[t][u] == -INFINITY ? 0.f : m[t][u];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = ex2(fmaf(v[e], a.c, -from));
        if (KEEP) l[t][u] += (v[0] + v[1]) + (v[2] + v[3]);
        p[t][u] = Half2<T>::pack(v[0], v[1]);
        p[t][2 + u] = Half2<T>::pack(v[2], v[3]);
        const float2 r0 = Half2<T>::unpack(p[t][u]), r1 = Half2<T>::unpack(p[t][2 + u]);
        w[t][u] += (r0.x + r0.y) + (r1.x + r1.y);
      }
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
      uint32_t vf[4];
      ldmatrix4t(row_addr<DP>(vt, mrow, n + mch), vf);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        mma16816<T>(o[t][n], p[t], vf[0], vf[1]);
        mma16816<T>(o[t][n + 1], p[t], vf[2], vf[3]);
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");

  // ---- join the four warps; lane (g, c) holds columns 8 n + 2c, + 1 of rows g and g + 8
  __syncthreads();                                         // the rings become the exchange buffer
  constexpr int LD = DP + 4;
  float* s_o = reinterpret_cast<float*>(smem_raw);
  float* mine = s_o + warp * 16 * MT * LD;
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (KEEP) {
        l[t][u] += __shfl_xor_sync(0xffffffffu, l[t][u], 1);
        l[t][u] += __shfl_xor_sync(0xffffffffu, l[t][u], 2);
      }
      w[t][u] += __shfl_xor_sync(0xffffffffu, w[t][u], 1);
      w[t][u] += __shfl_xor_sync(0xffffffffu, w[t][u], 2);
      const int lr = 16 * t + g + 8 * u;
      if (c == 0) {
        s_m[warp][lr] = m[t][u];
        if (KEEP) s_l[warp][lr] = l[t][u];
        s_w[warp][lr] = w[t][u];
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(mine + lr * LD + 8 * n + 2 * c) = make_float2(o[t][n][2 * u], o[t][n][2 * u + 1]);
    }
  __syncthreads();
  const int slot_out = split + (second ? a.seg[0].splits : 0);
  const long long qrows = (long long)a.B * a.Tq * a.H;
  const int per_row = a.D / 8, rows_here = min(16 * MT, s.R - row0);
  for (int i = threadIdx.x; i < rows_here * per_row; i += STEP_THREADS) {
    const int lr = i / per_row, d = (i - lr * per_row) * 8, r = row0 + lr;
    float big = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) big = fmaxf(big, s_m[i][lr]);
    const float from = big == -INFINITY ? 0.f : big;
    float sum = 0.f, weights = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = ex2(s_m[i][lr] - from);
      if (KEEP) sum += f * s_l[i][lr];
      weights += f * s_w[i][lr];
      const float* po = s_o + (i * 16 * MT + lr) * LD + d;
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] += f * po[k];
    }
    if (a.slots == 1) {
      write_row<T>(a, s, mem, hk, r, d, big, sum, weights, v);
    } else if (a.cluster) {
      // over the first warp's share, which only this thread still reads
      float* po = s_o + lr * LD + d;
#pragma unroll
      for (int k = 0; k < 8; ++k) po[k] = v[k];
      if (d == 0) {
        s_join[lr] = make_float2(big, weights);
        if (KEEP) s_join_l[lr] = sum;
      }
    } else {
      const long long qrow = query_row(a, s, mem, hk, r);
      float* po = a.part_o + ((long long)slot_out * qrows + qrow) * a.D + d;
      *reinterpret_cast<float4*>(po) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(po + 4) = make_float4(v[4], v[5], v[6], v[7]);
      if (d == 0) {
        a.part_mw[slot_out * qrows + qrow] = make_float2(big, weights);
        if (KEEP) a.part_l[slot_out * qrows + qrow] = sum;
      }
    }
  }
  if (a.cluster && a.slots > 1) {
    __syncwarp();
    // every block of the cluster has its part in shared memory; block b of n takes every n-th 8-column piece of the rows
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    const uint32_t o_at = smem_u32(s_o), j_at = smem_u32(s_join), l_at = smem_u32(s_join_l);
    for (int i = split * STEP_THREADS + threadIdx.x; i < rows_here * per_row; i += a.slots * STEP_THREADS) {
      const int lr = i / per_row, d = (i - lr * per_row) * 8;
      float big = -INFINITY, sum = 0.f, weights = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      float2 mw[8];
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        mw[b] = b < a.slots ? remote_float2(j_at + lr * 8, b) : make_float2(-INFINITY, 0.f);
        big = fmaxf(big, mw[b].x);
      }
      const float from = big == -INFINITY ? 0.f : big;
#pragma unroll
      for (int b = 0; b < 8; ++b)
        if (b < a.slots) {
          const float f = ex2(mw[b].x - from);
          weights += f * mw[b].y;
          if (KEEP && d == 0) sum += f * load_remote(in_block(l_at + lr * 4, b));
#pragma unroll
          for (int k = 0; k < 8; k += 2) {
            const float2 x = remote_float2(o_at + (lr * LD + d + k) * 4, b);
            v[k] += f * x.x;
            v[k + 1] += f * x.y;
          }
        }
      write_row<T>(a, s, mem, hk, row0 + lr, d, big, sum, weights, v);
    }
    __syncwarp();
    // no block leaves while another may still read its shared memory
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

// One warp per query row joins the parts of its blocks.
template <typename T> __global__ void __launch_bounds__(128) step_join_kernel(const StepArgs a) {
  const long long qrows = (long long)a.B * a.Tq * a.H, qrow = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (qrow >= qrows) return;
  const int lane = threadIdx.x & 31;
  float big = -INFINITY;
  for (int i = lane; i < a.slots; i += 32) big = fmaxf(big, a.part_mw[i * qrows + qrow].x);
  big = warp_max(big);
  const float base = big == -INFINITY ? 0.f : big;
  float sum = 0.f, weights = 0.f;
  for (int i = lane; i < a.slots; i += 32) {
    const float2 mw = a.part_mw[i * qrows + qrow];
    const float f = ex2(mw.x - base);
    weights += f * mw.y;
    if (a.lse) sum += f * a.part_l[i * qrows + qrow];
  }
  weights = warp_sum(weights);
  sum = warp_sum(sum);
  const float inv = weights == 0.f ? 0.f : 1.f / weights;
  if (4 * lane < a.D) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = 0; i < a.slots; ++i) {
      const float f = ex2(a.part_mw[i * qrows + qrow].x - base);
      const float4 p = *reinterpret_cast<const float4*>(a.part_o + (i * qrows + qrow) * a.D + 4 * lane);
      v.x += f * p.x; v.y += f * p.y; v.z += f * p.z; v.w += f * p.w;
    }
    uint32_t r0, r1;
    const uint32_t o0 = out_pair<T>(v.x * inv, v.y * inv, r0), o1 = out_pair<T>(v.z * inv, v.w * inv, r1);
    *reinterpret_cast<uint2*>(a.out + qrow * a.D + 4 * lane) = make_uint2(o0, o1);
    if (a.rest) *reinterpret_cast<uint2*>(a.rest + qrow * a.D + 4 * lane) = make_uint2(r0, r1);
  }
  if (a.lse && lane == 0) {
    const int h = (int)(qrow % a.H), t = (int)(qrow / a.H % a.Tq), b = (int)(qrow / a.H / a.Tq);
    const int G = a.seg[0].rows_per, hk = h / a.rep;
    const long long r = ((long long)(b % G) * a.rep + h % a.rep) * a.Tq + t;
    a.lse[((long long)(b / G) * a.Hk + hk) * a.seg[0].R + r] = sum > 0.f ? big + log2f(sum) : (sum == 0.f ? INFINITY : sum);
  }
}

// Row blocks per warp: two where a segment has more than 32 packed rows; up to there a second block of threads that reads the same keys
// from the L2 is faster than fewer and larger blocks for all (three to an SM, not two).
int row_blocks(const StepArgs& a) { return a.seg[0].R > 32 || a.seg[1].R > 32 ? 2 : 1; }

// Splits both segments' keys so that the blocks that fit the SMs at once get equal shares, of at most MAX_SHARE keys: beyond one wave, short
// shares keep the last wave short (and are what lengths far below the cache's size leave empty).  At least 64 keys, 16 per warp.
constexpr int MAX_SHARE = 512;
int plan(StepArgs& a, int memories0, int memories1) {
  const int rows = 16 * row_blocks(a);
  for (int i = 0; i < 2; ++i) a.seg[i].row_groups = (a.seg[i].R + rows - 1) / rows;
  const long long u0 = (long long)memories0 * a.Hk * a.seg[0].row_groups, u1 = memories1 ? (long long)memories1 * a.Hk * a.seg[1].row_groups : 0;
  const long long total = u0 * a.seg[0].size + u1 * a.seg[1].size;
  const long long wave = (long long)sb_num_sms() * (row_blocks(a) == 1 ? 3 : 2);      // blocks that run at once
  long long chunk = (total / wave + 63) / 64 * 64;
  chunk = chunk < 64 ? 64 : (chunk > MAX_SHARE ? MAX_SHARE : chunk);
  a.slots = 0;
  long long blocks = 0;
  for (int i = 0; i < 2; ++i) {
    Segment& s = a.seg[i];
    const long long units = i ? u1 : u0;
    s.splits = units ? (int)((s.size + chunk - 1) / chunk) : 0;
    // eight blocks of a cluster in one wave instead of more and a second kernel: 22 us instead of 25 for one row, 7500 keys, 8 heads
    if (!memories1 && s.splits > 8 && units >= 8 && units * 8 <= wave) s.splits = 8;
    s.chunk = s.splits ? (int)(((s.size + s.splits - 1) / s.splits + 63) / 64 * 64) : 64;
    if (units * s.splits > 0x7fffffffll) return SB_BAD_ARGUMENT;
    s.blocks = (int)(units * s.splits);
    blocks += s.blocks;
    a.slots += s.splits;
  }
  a.cluster = !memories1 && a.slots <= 8;
  return blocks > 0x7fffffffll ? SB_BAD_ARGUMENT : 0;
}

long long workspace(const StepArgs& a) {
  return a.slots <= 1 || a.cluster ? 0 : (long long)a.slots * a.B * a.Tq * a.H * (a.D + 3) * 4;
}

template <typename T, int DP, int MT> int launch_rows(const StepArgs& a, cudaStream_t stream) {
  const auto kernel = a.lse ? step_kernel<T, DP, MT, true> : step_kernel<T, DP, MT, false>;
  const int rc = sb_allow_smem((const void*)kernel, StepSmem<DP, MT>::BYTES);
  if (rc) return rc;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(a.seg[0].blocks + a.seg[1].blocks));
  config.blockDim = dim3(STEP_THREADS);
  config.dynamicSmemBytes = StepSmem<DP, MT>::BYTES;
  config.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)a.slots;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = a.cluster && a.slots > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}
template <typename T, int DP> int launch_step(const StepArgs& a, cudaStream_t stream) {
  const int rc = row_blocks(a) == 1 ? launch_rows<T, DP, 1>(a, stream) : launch_rows<T, DP, 2>(a, stream);
  if (rc || a.slots == 1 || a.cluster) return rc;
  const long long qrows = (long long)a.B * a.Tq * a.H;
  step_join_kernel<T><<<(unsigned)((qrows + 3) / 4), 128, 0, stream>>>(a);
  return (int)cudaGetLastError();
}

int run(StepArgs& a, int type, void* ws, cudaStream_t stream) {
  if (a.slots > 1 && !a.cluster) {
    if (!ws) return SB_BAD_ARGUMENT;
    a.part_o = (float*)ws;
    const long long rows = (long long)a.slots * a.B * a.Tq * a.H;
    a.part_mw = (float2*)(a.part_o + rows * a.D);
    a.part_l = (float*)(a.part_mw + rows);
  }
  if (type == 0) return a.D <= 64 ? launch_step<__nv_bfloat16, 64>(a, stream) : launch_step<__nv_bfloat16, 128>(a, stream);
  return a.D <= 64 ? launch_step<__half, 64>(a, stream) : launch_step<__half, 128>(a, stream);
}

Segment memory_segment(const SbCrossAttention* g) {
  Segment s = {};
  s.k = (const uint16_t*)g->k; s.v = (const uint16_t*)g->v;
  s.k_sb = g->k_sb; s.k_st = g->k_st; s.k_sh = g->k_sh;
  s.v_sb = g->v_sb; s.v_st = g->v_st; s.v_sh = g->v_sh;
  s.lengths = g->lengths; s.mask = g->mask;
  s.size = g->Tk; s.rows_per = g->G; s.causal = 0;
  s.R = g->G * g->rep * g->Tq;
  return s;
}

int fill(StepArgs& a, const SbCrossAttention* g) {
  XAttnArgs x;
  const int rc = sb_xattn_args(g, &x);
  if (rc) return rc;
  a = StepArgs{};
  a.q = (const uint16_t*)g->q;
  a.q_sb = g->q_sb; a.q_st = g->q_st; a.q_sh = g->q_sh;
  a.B = g->M * g->G; a.Tq = g->Tq; a.H = x.H; a.Hk = g->Hk; a.rep = g->rep; a.D = g->D;
  a.c = x.c;
  a.seg[0] = memory_segment(g);
  return 0;
}

}  // namespace

// Up to 32 packed rows.  [This kernel / the one for many rows, 8 heads of 128, us.  1 memory of 7500 keys: 1 row 23 / 25, 16 rows 27 / 29, 32
// rows 29 / 33, 64 rows 39 / 33; 16 of 500: 18 / 18, 23 / 23, 29 / 25, 41 / 25; 64 of 500: 41 / 55, 43 / 68, 49 / 78]
bool sb_few_rows(const SbCrossAttention* g) { return (long long)g->G * g->rep * g->Tq <= 32; }

int sb_step_cross_attention(const SbCrossAttention* g, void* out, void* rest, float* lse, void* ws, cudaStream_t stream) {
  StepArgs a;
  int rc = fill(a, g);
  if (rc) return rc;
  rc = plan(a, g->M, 0);
  if (rc) return rc;
  a.out = (uint16_t*)out;
  a.rest = (uint16_t*)rest;
  a.lse = lse;
  return run(a, g->type, ws, stream);
}

// Bytes of scratch memory that sb_cross_attention_fwd needs for this call; negative for invalid arguments.
SB_API long long sb_cross_attention_workspace(const SbCrossAttention* g) {
  StepArgs a;
  if (fill(a, g) || plan(a, g->M, 0)) return -1;
  return sb_few_rows(g) ? workspace(a) : 0;
}

// Own caches of a shared-prefix call; packed field by field in native_cross_attention.py.
struct SbOwnCache {
  const void *k, *v;
  long long k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  const int* lengths;
  int size, pad;
};

static int shared_prefix(StepArgs& a, const SbCrossAttention* g, const SbOwnCache* o) {
  int rc = fill(a, g);
  if (rc) return rc;
  if (!o || !o->k || !o->v || !o->lengths || o->size <= 0) return SB_BAD_ARGUMENT;
  if ((((uintptr_t)o->k | (uintptr_t)o->v) & 15) || o->k_sb % 8 || o->k_st % 8 || o->k_sh % 8 || o->v_sb % 8 || o->v_st % 8 || o->v_sh % 8)
    return SB_BAD_ARGUMENT;
  Segment& s = a.seg[1];
  s.k = (const uint16_t*)o->k; s.v = (const uint16_t*)o->v;
  s.k_sb = o->k_sb; s.k_st = o->k_st; s.k_sh = o->k_sh;
  s.v_sb = o->v_sb; s.v_st = o->v_st; s.v_sh = o->v_sh;
  s.lengths = o->lengths;
  s.size = o->size; s.rows_per = 1; s.causal = 1;
  s.R = g->rep * g->Tq;
  return plan(a, g->M, g->M * g->G);
}

SB_API long long sb_shared_prefix_workspace(const SbCrossAttention* g, const SbOwnCache* o) {
  StepArgs a;
  return shared_prefix(a, g, o) ? -1 : workspace(a);
}

SB_API int sb_shared_prefix_attention(const SbCrossAttention* g, const SbOwnCache* o, void* out, void* ws, cudaStream_t stream) {
  StepArgs a;
  const int rc = shared_prefix(a, g, o);
  if (rc) return rc;
  if (!out) return SB_BAD_ARGUMENT;
  a.out = (uint16_t*)out;
  return run(a, g->type, ws, stream);
}
