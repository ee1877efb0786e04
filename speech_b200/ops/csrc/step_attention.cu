// Attention for a few query rows per key head: one decoding step over an encoder's states, or over a prompt that a group of rows
// shares together with every row's own cache; also the forward pass of short queries in training.
//
// Keys and values are read once and little is computed on them, so bytes bound it, and what counts is how many loads are in flight:
// the keys of a (memory, key head) are split over blocks and over the warps of a block, every warp streams 16 keys at a time straight
// into registers in the fragment order of mma.m16n8k16, and the parts (running maximum m, sum l, unnormalised output) are joined in
// the block and, for more than one block, by a second small kernel:  o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.
//
// Fragment order without shared memory: a sum over d may take d in any order as long as both operands use the same one, so lane
// (g, c) = (lane / 4, lane % 4) reads 16 contiguous bytes (8 d) of key g and uses them as the k indices {2c, 2c+1, 2c+8, 2c+9} of two
// successive products; and a tile of 8 output columns may be any 8 d, so that lane reads 8 contiguous d of each of its four value
// rows and hands element j of them to output tile j.  All loads are whole 32-byte sectors, 16 bytes a lane.
//
// Sixteen packed rows (rows that read the same keys: group x heads of a key head x tokens, as in cross_attention.cuh) make a row
// block.  Up to four row blocks run in one block of threads, one per warp, so that the L1 serves their common keys; the rest of the
// four warps split the keys.
//
// Rounding: as in cross_attention_fwd.cu (weights rounded to 16 bits for the second product, all else fp32).
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
  int row_warps;            // warps of a block that take different row blocks
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
  uint16_t *out, *rest;     // [B, Tq, H, D]; rest: what rounding took from out, or null
  float* lse;               // packed rows of segment 0, or null
  float* part_o;            // [slots, B * Tq * H, D]
  float2* part_ml;          // [slots, B * Tq * H]
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

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ uint4 load16(const uint16_t* p, bool ok) {
  return ok ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
}

constexpr int STEP_THREADS = 128;

template <typename T, int DP>
__global__ void __launch_bounds__(STEP_THREADS, 3) step_kernel(const StepArgs a) {
  constexpr int KS = DP / 32, HV = DP / 64, NT = DP / 8;
  __shared__ float s_m[4][16], s_l[4][16];
  extern __shared__ float s_o[];                         // [4][16][DP + 4]
  const int second = blockIdx.x >= a.seg[0].blocks ? 1 : 0;
  const Segment& s = a.seg[second];
  int x = blockIdx.x - (second ? a.seg[0].blocks : 0);
  const int split = x % s.splits;
  x /= s.splits;
  const int rg = x % s.row_groups;
  x /= s.row_groups;
  const int hk = x % a.Hk, mem = x / a.Hk;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int row_warp = warp % s.row_warps, key_warp = warp / s.row_warps, key_warps = 4 / s.row_warps;
  const int row0 = (rg * s.row_warps + row_warp) * 16;

  int len = s.size;
  if (s.lengths) len = min(max(s.lengths[mem], 0), s.size);
  const int key_begin = split * s.chunk, key_end = min(len, key_begin + s.chunk);

  // packed row -> (batch row, token, head); rows g and g + 8 of the block
  int seen[2];
  uint4 q0[KS], q1[KS];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = row0 + g + 8 * u;
    const bool ok = r < s.R;
    const int y = r / a.Tq, t = r - y * a.Tq, gr = y / a.rep;
    const uint16_t* p = a.q + (long long)(mem * s.rows_per + gr) * a.q_sb + (long long)t * a.q_st + (long long)(hk * a.rep + y - gr * a.rep) * a.q_sh + 8 * c;
    seen[u] = !ok ? 0 : (s.causal ? len - a.Tq + 1 + t : len);
#pragma unroll
    for (int k = 0; k < KS; ++k) (u ? q1 : q0)[k] = load16(p + 32 * k, ok && 32 * k + 8 * c < a.D);
  }
  const uint16_t* kp = s.k + (long long)mem * s.k_sb + (long long)hk * s.k_sh + 8 * c;
  const uint16_t* vp = s.v + (long long)mem * s.v_sb + (long long)hk * s.v_sh + 8 * g;
  const uint8_t* mask = s.mask ? s.mask + (long long)mem * s.size : nullptr;

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

  uint4 kr[2][KS];
  auto load_keys = [&](int key0) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int key = key0 + 8 * n + g;
      const uint16_t* p = kp + (long long)key * s.k_st;
#pragma unroll
      for (int k = 0; k < KS; ++k) kr[n][k] = load16(p + 32 * k, key < key_end && 32 * k + 8 * c < a.D);
    }
  };
  int key0 = key_begin + key_warp * 16;
  if (row0 < s.R && key0 < key_end) load_keys(key0);
  for (; row0 < s.R && key0 < key_end; key0 += key_warps * 16) {
    // this lane's four keys, in score columns and in value rows alike: key0 + {2c, 2c+1, 2c+8, 2c+9}
    bool see[4];
    uint4 vr[4][HV];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = key0 + 2 * c + (i & 1) + 8 * (i >> 1);
      see[i] = key < key_end && !(mask && mask[key]);
      const uint16_t* p = vp + (long long)key * s.v_st;
#pragma unroll
      for (int h = 0; h < HV; ++h) vr[i][h] = load16(p + 64 * h, see[i] && 64 * h + 8 * g < a.D);   // a hidden value never meets its zero weight
    }
    float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const uint32_t a0[4] = {q0[k].x, q1[k].x, q0[k].y, q1[k].y}, a1[4] = {q0[k].z, q1[k].z, q0[k].w, q1[k].w};
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        mma16816<T>(sc[n], a0, kr[n][k].x, kr[n][k].y);
        mma16816<T>(sc[n], a1, kr[n][k].z, kr[n][k].w);
      }
    }
    if (key0 + key_warps * 16 < key_end) load_keys(key0 + key_warps * 16);
    uint32_t p[4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {                         // row g + 8 u: columns sc[n][2u], sc[n][2u + 1]
      float v[4];
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + 2 * c + (i & 1) + 8 * (i >> 1);
        v[i] = see[i] && key < seen[u] ? sc[i >> 1][2 * u + (i & 1)] * a.c : -INFINITY;
        mx = fmaxf(mx, v[i]);
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const bool grow = mx > m[u] + 8.f && m[u] != -INFINITY;
      if (__any_sync(0xffffffffu, grow)) {                // rare: the output keeps its scale until a maximum has grown by 2^8
        const float nm = m[u] == -INFINITY ? m[u] : fmaxf(m[u], mx);
        const float f = m[u] == -INFINITY ? 1.f : ex2(m[u] - nm);
        m[u] = nm;
        l[u] *= f;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          o[i][2 * u] *= f;
          o[i][2 * u + 1] *= f;
        }
      }
      if (m[u] == -INFINITY) m[u] = mx;
      const float base = m[u] == -INFINITY ? 0.f : m[u];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = ex2(v[i] - base);
      l[u] += (v[0] + v[1]) + (v[2] + v[3]);
      p[u] = Half2<T>::pack(v[0], v[1]);
      p[2 + u] = Half2<T>::pack(v[2], v[3]);
    }
#pragma unroll
    for (int h = 0; h < HV; ++h)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t sel = j & 1 ? 0x7632 : 0x5410;
        const uint32_t b0 = __byte_perm(word_of(vr[0][h], j >> 1), word_of(vr[1][h], j >> 1), sel);
        const uint32_t b1 = __byte_perm(word_of(vr[2][h], j >> 1), word_of(vr[3][h], j >> 1), sel);
        mma16816<T>(o[8 * h + j], p, b0, b1);
      }
  }
  // join the warps that split the keys of a row block; lane (g, c) holds, of rows g and g + 8, columns 64 h + 16 c + 0 .. 15
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
    l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
    if (c == 0) {
      s_m[warp][g + 8 * u] = m[u];
      s_l[warp][g + 8 * u] = l[u];
    }
  }
  constexpr int LD = DP + 4;
  float* mine = s_o + warp * 16 * LD;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int h = 0; h < HV; ++h)
#pragma unroll
      for (int n = 0; n < 2; ++n)                          // column 2c + n of tile j is d = 64 h + 8 (2c + n) + j
#pragma unroll
        for (int j = 0; j < 8; j += 4)
          *reinterpret_cast<float4*>(mine + (g + 8 * u) * LD + 64 * h + 16 * c + 8 * n + j) =
              make_float4(o[8 * h + j][2 * u + n], o[8 * h + j + 1][2 * u + n], o[8 * h + j + 2][2 * u + n], o[8 * h + j + 3][2 * u + n]);
  __syncthreads();
  const int slot = split + (second ? a.seg[0].splits : 0);
  const long long qrows = (long long)a.B * a.Tq * a.H;
  const int per_row = a.D / 8;
  for (int i = threadIdx.x; i < s.row_warps * 16 * per_row; i += STEP_THREADS) {
    const int rr = i / per_row, d = (i - rr * per_row) * 8, rw = rr >> 4, lr = rr & 15;
    const int r = (rg * s.row_warps + rw) * 16 + lr;
    if (r >= s.R) continue;
    float big = -INFINITY;
    for (int w = 0; w < key_warps; ++w) big = fmaxf(big, s_m[rw + w * s.row_warps][lr]);
    const float base = big == -INFINITY ? 0.f : big;
    float sum = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < key_warps; ++w) {
      const int src = rw + w * s.row_warps;
      const float f = ex2(s_m[src][lr] - base);
      sum += f * s_l[src][lr];
      const float* po = s_o + src * 16 * LD + lr * LD + d;
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] += f * po[k];
    }
    const int y = r / a.Tq, t = r - y * a.Tq, gr = y / a.rep;
    const long long qrow = ((long long)(mem * s.rows_per + gr) * a.Tq + t) * a.H + hk * a.rep + y - gr * a.rep;
    if (a.slots == 1) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      uint32_t o4[4], r4[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) o4[k] = out_pair<T>(v[2 * k] * inv, v[2 * k + 1] * inv, r4[k]);
      *reinterpret_cast<uint4*>(a.out + qrow * a.D + d) = make_uint4(o4[0], o4[1], o4[2], o4[3]);
      if (a.rest) *reinterpret_cast<uint4*>(a.rest + qrow * a.D + d) = make_uint4(r4[0], r4[1], r4[2], r4[3]);
      if (a.lse && d == 0) a.lse[((long long)mem * a.Hk + hk) * s.R + r] = sum > 0.f ? big + log2f(sum) : (sum == 0.f ? INFINITY : sum);
    } else {
      float* po = a.part_o + ((long long)slot * qrows + qrow) * a.D + d;
      *reinterpret_cast<float4*>(po) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(po + 4) = make_float4(v[4], v[5], v[6], v[7]);
      if (d == 0) a.part_ml[slot * qrows + qrow] = make_float2(big, sum);
    }
  }
}

// One warp per query row joins the parts of its blocks.
template <typename T> __global__ void __launch_bounds__(128) step_join_kernel(const StepArgs a) {
  const long long qrows = (long long)a.B * a.Tq * a.H, qrow = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (qrow >= qrows) return;
  const int lane = threadIdx.x & 31;
  float big = -INFINITY;
  for (int i = lane; i < a.slots; i += 32) big = fmaxf(big, a.part_ml[i * qrows + qrow].x);
  big = warp_max(big);
  const float base = big == -INFINITY ? 0.f : big;
  float sum = 0.f;
  for (int i = lane; i < a.slots; i += 32) {
    const float2 ml = a.part_ml[i * qrows + qrow];
    sum += ex2(ml.x - base) * ml.y;
  }
  sum = warp_sum(sum);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (4 * lane < a.D) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = 0; i < a.slots; ++i) {
      const float f = ex2(a.part_ml[i * qrows + qrow].x - base);
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

void plan_rows(Segment& s) {
  const int blocks16 = (s.R + 15) / 16;
  s.row_warps = blocks16 >= 4 ? 4 : (blocks16 >= 2 ? 2 : 1);
  s.row_groups = (blocks16 + s.row_warps - 1) / s.row_warps;
}

// Splits both segments' keys so that about three blocks per SM have equal shares.  A share is at least 64 keys (16 per warp).
int plan(StepArgs& a, int memories0, int memories1) {
  plan_rows(a.seg[0]);
  if (memories1) plan_rows(a.seg[1]);
  const long long u0 = (long long)memories0 * a.Hk * a.seg[0].row_groups, u1 = memories1 ? (long long)memories1 * a.Hk * a.seg[1].row_groups : 0;
  const long long total = u0 * a.seg[0].size + u1 * a.seg[1].size;
  long long chunk = (total / (148 * 3) + 63) / 64 * 64;
  if (chunk < 64) chunk = 64;
  a.slots = 0;
  long long blocks = 0;
  for (int i = 0; i < 2; ++i) {
    Segment& s = a.seg[i];
    const long long units = i ? u1 : u0;
    s.splits = units ? (int)((s.size + chunk - 1) / chunk) : 0;
    if (units && s.splits < 1) s.splits = 1;
    s.chunk = s.splits ? (int)(((s.size + s.splits - 1) / s.splits + 15) / 16 * 16) : 0;
    if (s.chunk < 16) s.chunk = 16;
    if (units * s.splits > 0x7fffffffll) return SB_BAD_ARGUMENT;
    s.blocks = (int)(units * s.splits);
    blocks += s.blocks;
    a.slots += s.splits;
  }
  return blocks > 0x7fffffffll ? SB_BAD_ARGUMENT : 0;
}

long long workspace(const StepArgs& a) {
  return a.slots <= 1 ? 0 : (long long)a.slots * a.B * a.Tq * a.H * (a.D + 2) * 4;
}

template <typename T, int DP> int launch_step(const StepArgs& a, cudaStream_t stream) {
  constexpr int SMEM = 4 * 16 * (DP + 4) * 4;
  step_kernel<T, DP><<<(unsigned)(a.seg[0].blocks + a.seg[1].blocks), STEP_THREADS, SMEM, stream>>>(a);
  int rc = (int)cudaGetLastError();
  if (rc || a.slots == 1) return rc;
  const long long qrows = (long long)a.B * a.Tq * a.H;
  step_join_kernel<T><<<(unsigned)((qrows + 3) / 4), 128, 0, stream>>>(a);
  return (int)cudaGetLastError();
}

int run(StepArgs& a, int type, void* ws, cudaStream_t stream) {
  if (a.slots > 1) {
    if (!ws) return SB_BAD_ARGUMENT;
    a.part_o = (float*)ws;
    a.part_ml = (float2*)(a.part_o + (long long)a.slots * a.B * a.Tq * a.H * a.D);
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

bool sb_few_rows(const SbCrossAttention* g) { return (long long)g->G * g->rep * g->Tq <= 64; }

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

// Own caches of a shared-prefix call; mirrored in native_cross_attention.py.
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
