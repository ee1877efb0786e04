// Losses of preference / policy optimisation straight from logits: clipped policy loss with a KL term, paired preference loss.
//
// For a row x (one position, V logits) with target y:   logp = x_y - m - log s,   m = max x,  s = sum exp(x - m)
//   policy      r = exp(logp - old),  term = -min(r A, clip(r) A) + beta (exp(d) - d - 1),  d = ref - logp
//               loss = sum_counted term / count,   slope = dloss/dlogp = (-r A [r A <= clip(r) A] + beta (1 - exp(d))) / count
//   preference  ratio_i = sum_counted (logp - ref) of sequence i,  margin = ratio_chosen - ratio_rejected, a scalar loss of the
//               margin per pair; slope of every counted position of a sequence = +-(dloss/dmargin) / pairs
//   gradient    dx_v = slope (1[v = y] - exp(x_v - m) / s)
//
// What bounds them: bytes.  The policy loss knows a row's slope as soon as it knows the row's logp, so the forward pass writes the
// gradient (for an upstream gradient of 1) while the row is still on the chip: logits are read from memory once.  A preference
// slope needs both sequences of the pair, so the rows are read a second time; the gradient kernel walks them backwards, and what
// the forward pass read last is then still in the L2.
//
// Rounding: exponentials are fp32 and so is a thread's share of a policy row's sum; shares are joined in fp64, and logp, the clip
// decision and the sums over rows are fp64: a policy at its reference has log ratios near zero, and in fp32 the rounding of a logp of
// -8 (5e-7) would be all that is left after a few thousand positions are summed.  A position's term and slope come from its fp64 log
// ratios in fp32, each a few units in its last place off.  For the same reason the preference loss has exponentials of its own, off by 4e-10 in
// the mean of many arguments (the library's moved every row's log sum the same way, by 1e-8, the approximate power of two by 7e-8, which a sum
// over a sequence multiplies and the mean of the policy loss does not), and rounds only the sums of four of them.  Its logarithm of the row's sum is
// the library's in fp64; the policy loss's is log s = k ln 2 + log f with s = 2^k f, f in [0.71, 1.42): the fp32 logarithm of f is off by less
// than 2^-24.  The gradient is rounded once.  Every sum has a fixed order (no floating-point atomics).
#include "packed_math.cuh"
#include <cuda_fp16.h>
#include <math.h>

namespace {

template <typename T> struct Vec;   // 16-byte groups of the logits' type
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      f[2 * u] = __uint_as_float(w[u] << 16);
      f[2 * u + 1] = __uint_as_float(w[u] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    __align__(16) __nv_bfloat162 o[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) o[u] = __floats2bfloat162_rn(f[2 * u], f[2 * u + 1]);
    return *reinterpret_cast<uint4*>(o);
  }
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
  using Max = __nv_bfloat162;
  static __device__ __forceinline__ Max lowest() { return __floats2bfloat162_rn(-INFINITY, -INFINITY); }
  static __device__ __forceinline__ Max max_of(Max m, const uint4& r) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
    return __hmax2(__hmax2(m, h[0]), __hmax2(h[1], __hmax2(h[2], h[3])));
  }
  static __device__ __forceinline__ float top(Max m) { return fmaxf(__low2float(m), __high2float(m)); }
  static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16(v); }
};
template <> struct Vec<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float2 v = __half22float2(h[u]);
      f[2 * u] = v.x;
      f[2 * u + 1] = v.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    __align__(16) __half2 o[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) o[u] = __floats2half2_rn(f[2 * u], f[2 * u + 1]);
    return *reinterpret_cast<uint4*>(o);
  }
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
  using Max = __half2;
  static __device__ __forceinline__ Max lowest() { return __floats2half2_rn(-INFINITY, -INFINITY); }
  static __device__ __forceinline__ Max max_of(Max m, const uint4& r) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
    return __hmax2(__hmax2(m, h[0]), __hmax2(h[1], __hmax2(h[2], h[3])));
  }
  static __device__ __forceinline__ float top(Max m) { return fmaxf(__low2float(m), __high2float(m)); }
  static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
};
template <> struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  using Max = float;
  static __device__ __forceinline__ Max lowest() { return -INFINITY; }
  static __device__ __forceinline__ Max max_of(Max m, const uint4& r) {
    return fmaxf(max3(m, __uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
  }
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  static __device__ __forceinline__ float top(Max m) { return m; }
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
};

// n / d for 0 <= n < 2^31 and a divisor known on the host: the high half of n * (2^(31 + s) / d + 1), s the bits of d - 1.
struct Divisor {
  uint32_t mul;
  int shift;                        // -1: d = 1
};
inline Divisor divisor(int d) {
  if (d == 1) return {0, -1};
  int s = 1;
  while ((1ll << s) < d) ++s;
  return {(uint32_t)((1ull << (31 + s)) / (unsigned)d + 1), s - 1};
}
__device__ __forceinline__ int divide(int n, Divisor d) { return d.shift < 0 ? n : (int)(__umulhi((uint32_t)n, d.mul) >> d.shift); }

struct RowArgs {
  const void* logits;               // row (n, t, c) starts at element n * sn + t * st + c * sc
  long long sn, st, sc;
  const long long* targets;         // [rows]
  const uint8_t* mask;              // [N * T], null = every position counts
  const float* ref;                 // [rows] or null
  const float* old;                 // [rows] or null
  const float* adv;                 // [N]
  int rows;
  int T, C, V;
  Divisor by_c, by_t;
  float clip_lo, clip_hi, kl_beta;
  double log_lo, log_hi;             // log(1 - clip_lo), log(1 + clip_hi): the clip decision is taken on log ratios
};

struct Row { int n, nt; long long off; };
__device__ __forceinline__ Row locate(const RowArgs& a, int row) {
  Row r;
  r.nt = divide(row, a.by_c);
  r.n = divide(r.nt, a.by_t);
  r.off = r.n * a.sn + (r.nt - r.n * a.T) * a.st + (row - r.nt * a.C) * a.sc;
  return r;
}

// The 16-byte groups of a row start at its first aligned element: `head` elements before it and `tail` after the last whole group
// are handled one by one (a row of an odd number of 16-bit logits starts at any even address).
struct Span { int head, nv, tail; };
template <typename T> __device__ __forceinline__ Span span_of(const T* p, int V) {
  Span s;
  s.head = (int)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T));
  if (s.head > V) s.head = V;
  s.nv = (V - s.head) / Vec<T>::N;
  s.tail = V - s.head - s.nv * Vec<T>::N;
  return s;
}

// (max, sum) pairs with sum taken relative to max; an empty share is (-inf, 0)
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

constexpr float LOG2E = 1.44269504f;
enum { LOSS_POLICY = 0, LOSS_PREFERENCE = 1 };

// exp of two values t <= 0 (above 88 the exponent's bits overflow), off by less than 0.6 units in the last place and, in the mean of many
// arguments, by 4e-10 (of the few differences that bf16 logits have, by up to 4e-9: rewards of 2 x 512 rows of 40001, 3.4e-9 a row):
// t log2 e = n + f with n the nearest integer (what adding 1.5 * 2^23 leaves) and f from the product with log2 e in two parts, after Cody and Waite
// (Software Manual for the Elementary Functions, 1980); 2^f = 1 + f q(f), q of degree 5 through
// (2^f - 1) / f at the six Chebyshev nodes of [-1/2, 1/2]; times 2^n.  Below e^-88 the result is 0; NaN stays NaN.
__device__ __forceinline__ uint64_t exp_fine(uint64_t v) {
  float t, u;
  split(v, t, u);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(t) : "f"(-88.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(u) : "f"(-88.f));
  const uint64_t x = pair(t, u);
  constexpr float ROUND = 12583039.f;                      // 1.5 * 2^23 + 127: the low bits of the sum are n + 127
  const uint64_t r = fma2(x, pair(1.44269502f, 1.44269502f), pair(ROUND, ROUND));
  uint64_t f = fma2(x, pair(1.44269502f, 1.44269502f), fma2(r, pair(-1.f, -1.f), pair(ROUND, ROUND)));
  f = fma2(x, pair(1.92596303e-8f, 1.92596303e-8f), f);
  uint64_t p = fma2(f, pair(0.00015453163f, 0.00015453163f), pair(0.0013390863f, 0.0013390863f));
  p = fma2(p, f, pair(0.009618083f, 0.009618083f));
  p = fma2(p, f, pair(0.05550357f, 0.05550357f));
  p = fma2(p, f, pair(0.2402265f, 0.2402265f));
  p = fma2(p, f, pair(0.6931472f, 0.6931472f));
  p = fma2(p, f, pair(1.f, 1.f));
  split(r, t, u);
  return mul2(p, pair(__float_as_uint(t) << 23, __float_as_uint(u) << 23));
}
__device__ __forceinline__ float exp_fine(float t) {
  float a, b;
  split(exp_fine(pair(t, t)), a, b);
  return a;
}

// A share of a row's sum, taken relative to m, relative to `base` >= m instead.  A share that has met no logit above -inf (m = -inf) stays as it
// is, zero or NaN: its factor would be exp of 0 - base, which is infinite or worse where base is below -88.
template <typename S> __device__ __forceinline__ S rebased(S share, float m, float base) {
  return m == -INFINITY ? share : share * (S)exp_fine(m - base);
}

// Softmax weight of a logit, 2^((x - m) log2 e - log2 s), from the row's m and log s.  Kept apart: in a row of nothing but the type's
// lowest value (a vocabulary masked wholly), m + log s would be m.
struct Weight {
  float m, shift;
  __device__ __forceinline__ explicit Weight(float2 lse) : m(lse.x), shift(-lse.y * LOG2E) {}
  __device__ __forceinline__ float operator()(float x) const { return ex2(fmaf(x - m, LOG2E, shift)); }
};

// exp(f - base), the even elements of a group of E summed in one half, the odd ones in the other
template <int E> __device__ __forceinline__ uint64_t exp_sum(const float* f, uint64_t shift2) {
  uint64_t e[E / 2];
#pragma unroll
  for (int u = 0; u < E / 2; ++u) e[u] = exp_fine(add2(pair(f[2 * u], f[2 * u + 1]), shift2));
  return E == 8 ? add2(add2(e[0], e[1]), add2(e[E / 2 - 2], e[E / 2 - 1])) : add2(e[0], e[1]);
}

// A sum of terms in [0, 4] without rounding: the sum is 4 at the start and thus never below a term, what an addition rounds away is
// then (term - (new sum - old sum)) exactly, and is summed beside it.
struct FineSum {
  uint64_t hi = pair(4.f, 4.f), lo = 0;
  __device__ __forceinline__ void add(uint64_t v) {
    const uint64_t t = add2(hi, v);
    lo = add2(lo, add2(v, fma2(t, pair(-1.f, -1.f), hi)));
    hi = t;
  }
  __device__ __forceinline__ double take() {
    float a, b, c, d;
    split(hi, a, b);
    split(lo, c, d);
    hi = pair(4.f, 4.f);
    lo = 0;
    return (((double)a - 4.0) + ((double)b - 4.0)) + ((double)c + (double)d);
  }
};

// A thread's share of a row's sum: fp32, or fp64 where the rows' logarithms are summed in turn.
template <int MODE> struct SumOf { using type = float; };
template <> struct SumOf<LOSS_PREFERENCE> { using type = double; };
template <int MODE> using Sum = typename SumOf<MODE>::type;

// Joins the (max, sum) shares of the TPR threads of a row: one warp (TPR = 32) or a whole block.
template <int TPR, typename S> __device__ __forceinline__ void join(float& m, double& sum, S share, float* redf, double* redd) {
  const float wm = warp_max(m);
  double v = rebased((double)share, m, wm);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (TPR == 32) {
    m = finite_or_zero(wm);
    sum = v;
    return;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    redf[threadIdx.x >> 5] = wm;
    redd[threadIdx.x >> 5] = v;
  }
  __syncthreads();
  float bm = redf[0];
#pragma unroll
  for (int i = 1; i < TPR / 32; ++i) bm = fmaxf(bm, redf[i]);
  m = finite_or_zero(bm);
  sum = 0.0;
#pragma unroll
  for (int i = 0; i < TPR / 32; ++i) sum += rebased(redd[i], redf[i], m);
}

// exp(d) - 1 - d, to a few units in the last place: near zero by its Taylor series d^2 (1/2! + d/3! + ... + d^7/9!), because the difference
// of two numbers near d has their rounding (1e-4 of the term at d = 1e-3).  The series' rest is below 2^-24 of it for |d| <= 1/2.
__device__ __forceinline__ float expm1_beyond(float d) {
  if (fabsf(d) > 0.5f) return expm1f(d) - d;
  float p = 1.f / 362880.f;
  p = fmaf(p, d, 1.f / 40320.f);
  p = fmaf(p, d, 1.f / 5040.f);
  p = fmaf(p, d, 1.f / 720.f);
  p = fmaf(p, d, 1.f / 120.f);
  p = fmaf(p, d, 1.f / 24.f);
  p = fmaf(p, d, 1.f / 6.f);
  p = fmaf(p, d, 0.5f);
  return p * d * d;
}

__device__ __forceinline__ double log_of_sum(double s) {
  // s = 2^k f; also right for 0 (-inf), infinity and NaN, which the scaling leaves alone
  if (!(s > 1e-30 && s < 1e30)) return (double)logf((float)s);
  const float f = (float)s;
  int k = ((__float_as_int(f) - 0x3f350000) >> 23);
  const double scaled = s * __longlong_as_double((long long)(1023 - k) << 52);
  return (double)k * 0.693147180559945309417 + (double)logf((float)scaled);
}

template <typename T> __device__ __forceinline__ T* out_row(void* d, int row, int V) { return reinterpret_cast<T*>(d) + (long long)row * V; }

template <typename T, int TPR> __device__ __forceinline__ void write_zeros(T* o, int V, int lane) {
  const Span s = span_of(o, V);
  if (lane < s.head) o[lane] = Vec<T>::down(0.f);
  uint4* ov = reinterpret_cast<uint4*>(o + s.head);
  for (int i = lane; i < s.nv; i += TPR) ov[i] = make_uint4(0, 0, 0, 0);
  if (lane < s.tail) o[s.head + s.nv * Vec<T>::N + lane] = Vec<T>::down(0.f);
}

// Gradient of a row read again from memory: slope * (1[v = y] - exp(x - m) / s).  Input and output may be aligned differently
// (logits that are a slice of a longer tensor): groups are formed on the output where the input allows it, else one by one.
// The thread that wrote the target's element writes it once more, with its 1.
template <typename T, int TPR, int NV>
__device__ __forceinline__ void grad_from_memory(const T* x, T* o, int V, int lane, int y, float slope, float2 lse) {
  const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(o)) & 15) == 0;
  const Weight weight(lse);
  const float k = -slope;
  auto one = [&](int v) { o[v] = Vec<T>::down(fmaf(k, weight(Vec<T>::up(x[v])), v == y ? slope : 0.f)); };
  if (!same) {
    for (int v = lane; v < V; v += TPR) one(v);
    return;
  }
  constexpr int E = Vec<T>::N;
  const Span s = span_of(x, V);
  if (lane < s.head) one(lane);
  if (lane < s.tail) one(s.head + s.nv * E + lane);
  const uint4* xv = reinterpret_cast<const uint4*>(x + s.head);
  uint4* ov = reinterpret_cast<uint4*>(o + s.head);
  const uint64_t k2 = pair(k, k);
  for (int i0 = lane; i0 < s.nv; i0 += NV * TPR) {           // NV groups are read before the first is worked on
    uint4 raw[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (i0 + j * TPR < s.nv) raw[j] = xv[i0 + j * TPR];
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (i0 + j * TPR < s.nv) {
        float f[E];
        Vec<T>::unpack(raw[j], f);
#pragma unroll
        for (int u = 0; u < E; u += 2) split(mul2(pair(weight(f[u]), weight(f[u + 1])), k2), f[u], f[u + 1]);
        __stcs(ov + i0 + j * TPR, Vec<T>::pack(f));
      }
  }
  const int yv = y - s.head;
  if (yv >= 0 && yv < s.nv * E && (yv / E) % TPR == lane) one(y);
}

// Counted positions, by a whole block.  Every block counts for itself up to this many bytes of mask (a few loads per thread); beyond,
// a kernel does it first.
constexpr long long COUNT_LIMIT = 64 * 1024;
__device__ int count_mask(const uint8_t* __restrict__ mask, long long rows, int C, int* red) {
  if (!mask) return (int)rows;
  const long long nt = rows / C;
  int n = 0;
  const long long head = min(nt, (long long)((16 - (reinterpret_cast<uintptr_t>(mask) & 15)) & 15)), groups = (nt - head) / 16;
  if (threadIdx.x < head) n += mask[threadIdx.x] != 0;
  const uint4* g = reinterpret_cast<const uint4*>(mask + head);
  for (long long i = threadIdx.x; i < groups; i += blockDim.x) {
    const uint4 v = g[i];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) n += __popc(__vsetne4(w[k], 0u));
  }
  for (long long i = head + groups * 16 + threadIdx.x; i < nt; i += blockDim.x) n += mask[i] != 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = n;
  __syncthreads();
  int t = 0;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) t += red[i];
  __syncthreads();
  return t * C;
}

__device__ __forceinline__ void copy_async(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}

// Forward pass over all rows.  TPR threads work on a row; NV > 0: it stays in registers as it was read, NV 16-byte groups per thread;
// NV = 0: rows of any length, read again for the gradient, from the L2 (148 rows of 300 KB in flight are a third of it).
// lse: (m, log s) fp32 [rows]; logp / slope: fp32 [rows]; dlogits: contiguous [rows, V] or null (no gradient wanted now); partial:
// fp64, per block the sum of its policy terms; ratio: fp64 [rows], preference only.
// [110080 rows of 2024, bf16, with the gradient: 199 us with the row read as it is needed, 186 us a row ahead and without branches around
// its groups; 16 / 20 / 24 warps per SM: 186 / 246 / 281 us (spills).  27520 rows without a gradient: 16 / 20 / 24 warps 51 / 49 / 47 us.]
template <int MODE, int TPR> constexpr int resident_warps() { return TPR == 32 && MODE == LOSS_POLICY ? 16 : TPR == 32 || TPR == 256 ? 24 : 32; }
template <typename T, int MODE, int TPR, int NV, int THREADS, bool COUNT_HERE>
__global__ void __launch_bounds__(THREADS, resident_warps<MODE, TPR>() * 32 / THREADS)
rows_forward_kernel(const RowArgs a, int* __restrict__ count_p, float* __restrict__ logp_out, float2* __restrict__ lse_out, float* __restrict__ slope_out,
                    void* __restrict__ dlogits, double* __restrict__ partial, double* __restrict__ ratio) {
  constexpr int E = Vec<T>::N, GROUPS = THREADS / TPR;
  __shared__ float redf[32];
  __shared__ double redd[32];
  const int lane = TPR == 32 ? (threadIdx.x & 31) : threadIdx.x;
  const int group = TPR == 32 ? (threadIdx.x >> 5) : 0;
  int count = 0;
  if (MODE == LOSS_POLICY) count = COUNT_HERE ? count_mask(a.mask, a.rows, a.C, reinterpret_cast<int*>(redf)) : *count_p;
  const float inv_count = (float)(1.0 / (double)max(1, count));
  if (COUNT_HERE && blockIdx.x == 0 && threadIdx.x == 0) *count_p = count;
  double mine = 0.0;                                     // same value in every thread of the group
  const int step = gridDim.x * GROUPS;
  // A row's mask, target and log-probabilities are read two rows ahead; where a warp has a row to itself, the row follows one ahead, by
  // asynchronous copies into shared memory, each thread for itself, so that no latency stands between rows.
  constexpr bool AHEAD = TPR == 32;
  __shared__ uint4 copy[AHEAD ? NV * THREADS : 1];
  struct Ahead {
    uint8_t shown;                                       // a counted row
    long long off, y64;
    float old, ref, adv;
  };
  auto look = [&](int row) {                             // loads alone: what they bring is looked at a row later
    Ahead q = {0, 0, -1, 0.f, 0.f, 0.f};
    if (row < a.rows) {
      const Row r = locate(a, row);
      q.shown = a.mask ? a.mask[r.nt] : 1;
      q.off = r.off;
      q.y64 = a.targets[row];
      if (MODE == LOSS_POLICY) {
        q.old = a.old[row];
        q.adv = a.adv[r.n];
      }
      if (a.ref) q.ref = a.ref[row];
    }
    return q;
  };
  struct Edge { float hx, tx, xy; };                     // elements around the whole groups, the target's logit
  auto fetch = [&](const Ahead& q) {
    Edge e = {-INFINITY, -INFINITY, NAN};
    if (q.shown) {                                       // a hidden position's logits are not read
      const T* x = reinterpret_cast<const T*>(a.logits) + q.off;
      const Span s = span_of(x, a.V);
      const uint4* xv = reinterpret_cast<const uint4*>(x + s.head);
      if (AHEAD) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
          if (lane + k * TPR < s.nv) copy_async(copy + k * THREADS + threadIdx.x, xv + lane + k * TPR);
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
      if (q.y64 >= 0 && q.y64 < a.V) e.xy = Vec<T>::up(x[q.y64]);   // a target outside the vocabulary makes the row's results NaN
      if (lane < s.head) e.hx = Vec<T>::up(x[lane]);
      if (lane < s.tail) e.tx = Vec<T>::up(x[s.head + s.nv * E + lane]);
    }
    return e;
  };
  Edge edge_next;
  auto work = [&](int row, const Ahead& q, const Ahead& next, Edge edge) {
    T* o = dlogits ? out_row<T>(dlogits, row, a.V) : nullptr;
    if (!q.shown) {
      if (lane == 0) {
        lse_out[row] = make_float2(0.f, 0.f);
        if (MODE == LOSS_POLICY) logp_out[row] = slope_out[row] = 0.f;
        else ratio[row] = 0.0;
      }
      if (o) write_zeros<T, TPR>(o, a.V, lane);
      if (AHEAD) edge_next = fetch(next);
      return;
    }
    const T* x = reinterpret_cast<const T*>(a.logits) + q.off;
    const Span s = span_of(x, a.V);
    const uint4* xv = reinterpret_cast<const uint4*>(x + s.head);
    const int vt = s.head + s.nv * E, y = q.y64 >= 0 && q.y64 < a.V ? (int)q.y64 : -1;
    uint4 raw[NV > 0 ? NV : 1];
    if (AHEAD) asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      raw[k] = Vec<T>::none();                           // -inf: no part in the maximum and the sum, and no branch around them
      if (lane + k * TPR < s.nv) raw[k] = AHEAD ? copy[k * THREADS + threadIdx.x] : __ldcs(xv + lane + k * TPR);
    }
    if (!AHEAD) edge = fetch(q);
    const float hx = edge.hx, tx = edge.tx, xy = edge.xy, old = q.old, ref = q.ref, A = q.adv;
    float m = fmaxf(hx, tx);
    Sum<MODE> share;
    FineSum fine;
    float base = 0.f;
    auto edges = [&](float base) {
      if (MODE == LOSS_POLICY) return ex2((hx - base) * LOG2E) + ex2((tx - base) * LOG2E);
      float h, t;
      split(exp_fine(pair(hx - base, tx - base)), h, t);
      return h + t;
    };
    if (NV > 0) {
      typename Vec<T>::Max top = Vec<T>::lowest();
#pragma unroll
      for (int k = 0; k < NV; ++k) top = Vec<T>::max_of(top, raw[k]);
      m = fmaxf(m, Vec<T>::top(top));
      if (AHEAD) edge_next = fetch(next);                 // the values above are in registers: their place is free
      base = finite_or_zero(m);
      share = edges(base);
      const uint64_t scale2 = pair(LOG2E, LOG2E), shift2 = pair(-base, -base);
      uint64_t sum2[2] = {0, 0};
#pragma unroll
      for (int k = 0; k < NV; ++k) {
          float f[E];
          Vec<T>::unpack(raw[k], f);
          if (MODE == LOSS_POLICY) {
#pragma unroll
            for (int u = 0; u < E; u += 2) {
              float x, y;
              split(mul2(add2(pair(f[u], f[u + 1]), shift2), scale2), x, y);
              sum2[(u >> 1) & 1] = add2(sum2[(u >> 1) & 1], pair(ex2(x), ex2(y)));
            }
          } else {
            fine.add(exp_sum<E>(f, shift2));
          }
      }
      if (MODE == LOSS_POLICY) {
        float x, y;
        split(add2(sum2[0], sum2[1]), x, y);
        share += x + y;
      } else {
        share += fine.take();
      }
    } else {
      share = edges(finite_or_zero(m));
      constexpr int U = 4;
      uint4 now[U], later[U];
      auto read = [&](int i, uint4* to) {
#pragma unroll
        for (int k = 0; k < U; ++k) {
          to[k] = Vec<T>::none();
          if (i + k * TPR < s.nv) to[k] = xv[i + k * TPR];
        }
      };
      read(lane, later);
      for (int i = lane; i < s.nv; i += U * TPR) {
        typename Vec<T>::Max top = Vec<T>::lowest();
#pragma unroll
        for (int k = 0; k < U; ++k) {
          now[k] = later[k];
          top = Vec<T>::max_of(top, now[k]);
        }
        read(i + U * TPR, later);
        const float nm = fmaxf(m, Vec<T>::top(top));
        base = finite_or_zero(nm);
        if (nm > m) {                                    // rare after the first groups
          if (MODE == LOSS_PREFERENCE) share += fine.take();
          share = rebased(share, m, base);
          m = nm;
        }
        const uint64_t shift2 = pair(-base, -base);
#pragma unroll
        for (int k = 0; k < U; ++k) {
          float f[E];
          Vec<T>::unpack(now[k], f);
          if (MODE == LOSS_POLICY) {
#pragma unroll
            for (int u = 0; u < E; u += 2) {
              split(mul2(add2(pair(f[u], f[u + 1]), shift2), pair(LOG2E, LOG2E)), f[u], f[u + 1]);
              share += ex2(f[u]) + ex2(f[u + 1]);
            }
          } else {
            fine.add(exp_sum<E>(f, shift2));
          }
        }
      }
      if (MODE == LOSS_PREFERENCE) share += fine.take();
    }
    double sum;
    join<TPR>(m, sum, share, redf, redd);
    const double log_sum = MODE == LOSS_PREFERENCE ? log(sum) : log_of_sum(sum);
    const double logp = (double)xy - (double)m - log_sum;
    float slope = 0.f;
    if (MODE == LOSS_POLICY) {
      const double d = logp - (double)old;
      const float plain = expf((float)d) * A;
      const bool above = A > 0.f && d > a.log_hi, below = A < 0.f && d < a.log_lo;   // NaN is neither
      float each = above ? -(1.f + a.clip_hi) * A : below ? -(1.f - a.clip_lo) * A : -plain;
      slope = above || below ? 0.f : -plain;
      if (a.ref && a.kl_beta != 0.f) {
        const float kd = (float)((double)ref - logp);
        slope -= a.kl_beta * expm1f(kd);
        each += a.kl_beta * expm1_beyond(kd);
      }
      mine += (double)each;
      slope *= inv_count;
    }
    if (lane == 0) {
      lse_out[row] = make_float2(m, (float)log_sum);
      if (MODE == LOSS_POLICY) {
        logp_out[row] = (float)logp;
        slope_out[row] = slope;
      } else {
        ratio[row] = logp - (double)ref;
      }
    }
    if (MODE == LOSS_POLICY && o) {
      if (slope == 0.f) {
        write_zeros<T, TPR>(o, a.V, lane);
        return;
      }
      const float inv = 1.f / (float)sum;
      if (NV > 0 && ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(o)) & 15) == 0) {
        // from the registers as they were read: keeping the exponentials instead (64 more) halves the rows in flight, 250 us for 190
        const float k0 = -slope * inv;
        const uint64_t k2 = pair(k0, k0), l2 = pair(LOG2E, LOG2E), m2 = pair(-m, -m);
        auto put = [&](int v, float xf) { o[v] = Vec<T>::down(fmaf(k0, ex2((xf - m) * LOG2E), v == y ? slope : 0.f)); };
        uint4* ov = reinterpret_cast<uint4*>(o + s.head);
        if (lane < s.head) put(lane, hx);
        if (lane < s.tail) put(vt + lane, tx);
#pragma unroll
        for (int k = 0; k < NV; ++k)
          {
            float f[E];
            Vec<T>::unpack(raw[k], f);
#pragma unroll
            for (int u = 0; u < E; u += 2) {
              split(mul2(add2(pair(f[u], f[u + 1]), m2), l2), f[u], f[u + 1]);
              split(mul2(pair(ex2(f[u]), ex2(f[u + 1])), k2), f[u], f[u + 1]);
            }
            if (lane + k * TPR < s.nv) __stcs(ov + lane + k * TPR, Vec<T>::pack(f));
          }
        const int yv = y - s.head;                        // the target's element once more, by the thread that wrote its group
        if (yv >= 0 && yv < s.nv * E && (yv / E) % TPR == lane) put(y, xy);
      } else {
        grad_from_memory<T, TPR, 4>(x, o, a.V, lane, y, slope, make_float2(m, (float)log_sum));
      }
    }
  };
  int row = blockIdx.x * GROUPS + group;
  if (AHEAD) {
    Ahead cur = look(row), next = look(row + step);
    Edge edge = fetch(cur);
    for (; row < a.rows; row += step) {
      const Ahead after = look(row + 2 * step);
      work(row, cur, next, edge);
      cur = next;
      next = after;
      edge = edge_next;
    }
  } else {
    for (; row < a.rows; row += step) {
      const Ahead cur = look(row);
      work(row, cur, cur, Edge());
    }
  }
  if (MODE == LOSS_POLICY) {
    // fixed order: groups of the block in turn, blocks in turn (policy_finish_kernel)
    __syncthreads();
    if (TPR == 32) {
      if (lane == 0) redd[group] = mine;
      __syncthreads();
      if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < GROUPS; ++i) t += redd[i];
        partial[blockIdx.x] = t;
      }
    } else if (threadIdx.x == 0) {
      partial[blockIdx.x] = mine;
    }
  }
}

// Gradient of all rows from memory: per-row slopes (slope != null), or one slope per sequence with masked rows zero.  `upstream`
// is the gradient of the loss, in device memory; with `unless_one` the whole kernel has nothing to do when it is 1, which is what
// the forward pass has written the gradient for already.  Rows are walked from the last to the first.
template <typename T, int TPR, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS) rows_grad_kernel(const RowArgs a, const float2* __restrict__ lse, const float* __restrict__ slope,
                                                            const float* __restrict__ seq_slope, const float* __restrict__ upstream, int unless_one,
                                                            void* __restrict__ dlogits) {
  const float g = *upstream;
  if (unless_one && g == 1.f) return;
  constexpr int GROUPS = THREADS / TPR;
  const int lane = TPR == 32 ? (threadIdx.x & 31) : threadIdx.x;
  const int group = TPR == 32 ? (threadIdx.x >> 5) : 0;
  for (int i = blockIdx.x * GROUPS + group; i < a.rows; i += gridDim.x * GROUPS) {
    const int row = a.rows - 1 - i;
    const Row r = locate(a, row);
    T* o = out_row<T>(dlogits, row, a.V);
    const bool hidden = a.mask && !a.mask[r.nt];
    const float sl = hidden ? 0.f : g * (slope ? slope[row] : seq_slope[r.n]);
    if (sl == 0.f) {
      write_zeros<T, TPR>(o, a.V, lane);
      continue;
    }
    const long long y64 = a.targets[row];
    const int y = y64 >= 0 && y64 < a.V ? (int)y64 : -1;
    grad_from_memory<T, TPR, NV>(reinterpret_cast<const T*>(a.logits) + r.off, o, a.V, lane, y, sl, lse[row]);
  }
}

__global__ void __launch_bounds__(1024) count_kernel(const uint8_t* __restrict__ mask, long long rows, int C, int* __restrict__ count) {
  __shared__ int red[32];
  const int n = count_mask(mask, rows, C, red);
  if (threadIdx.x == 0) *count = n;
}

__global__ void __launch_bounds__(1024) policy_finish_kernel(const double* __restrict__ partial, int n, const int* __restrict__ count, float* __restrict__ loss) {
  __shared__ double red[32];
  double t = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += blockDim.x) t += partial[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    double u = 0.0;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) u += red[i];
    *loss = (float)(u / (double)max(1, *count));
  }
}

// One block per sequence: ratio_i = sum of its rows' log ratios.
__global__ void ratio_kernel(const double* __restrict__ ratio, long long per, double* __restrict__ total) {
  __shared__ double red[32];
  const double* p = ratio + (long long)blockIdx.x * per;
  double t = 0.0;
  for (long long i = threadIdx.x; i < per; i += blockDim.x) t += p[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    double u = 0.0;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) u += red[i];
    total[blockIdx.x] = u;
  }
}

// The same sums by one warp per sequence, in the block that goes on with them: for up to this many positions in all one kernel less is
// worth more than the wider sum.
constexpr long long ONE_BLOCK_ROWS = 64 * 1024;
__device__ void ratio_sums(const double* __restrict__ ratio, long long per, int n, double* total) {
  for (int s = threadIdx.x >> 5; s < n; s += blockDim.x >> 5) {
    const double* p = ratio + (long long)s * per;
    double t[4] = {0.0, 0.0, 0.0, 0.0};
    long long i = threadIdx.x & 31;
    for (; i + 96 < per; i += 128) {
#pragma unroll
      for (int k = 0; k < 4; ++k) t[k] += p[i + 32 * k];
    }
    for (; i < per; i += 32) t[0] += p[i];
    double u = (t[0] + t[1]) + (t[2] + t[3]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
    if ((threadIdx.x & 31) == 0) total[s] = u;
  }
  __syncthreads();
}

// Scalar losses of all pairs, their mean, rewards beta * ratio and the slope of every sequence's positions.  One block.
__global__ void __launch_bounds__(1024)
preference_finish_kernel(const double* __restrict__ ratio, long long per, double* total, int pairs, int kind, float beta_f, const float* __restrict__ gap,
                         float* __restrict__ loss, float* __restrict__ rewards, float* __restrict__ seq_slope) {
  __shared__ double red[32];
  const double beta = (double)beta_f;
  double mine = 0.0;
  if (ratio) ratio_sums(ratio, per, 2 * pairs, total);
  for (int n = threadIdx.x; n < pairs; n += blockDim.x) {
    const double margin = total[n] - total[n + pairs];
    double l, s;
    if (kind == 0) {                                        // -log sigmoid(beta margin)
      const double z = beta * margin;
      l = log1p(exp(-fabs(z))) + (z < 0.0 ? -z : 0.0);
      s = -beta / (1.0 + exp(z));
    } else if (kind == 1) {
      const double d = margin - 1.0 / (2.0 * beta);
      l = d * d;
      s = 2.0 * d;
    } else {
      const double d = beta * margin - (double)gap[n];
      l = d * d;
      s = 2.0 * beta * d;
    }
    mine += l;
    seq_slope[n] = (float)(s / pairs);
    seq_slope[n + pairs] = (float)(-s / pairs);
    rewards[n] = (float)(beta * total[n]);
    rewards[n + pairs] = (float)(beta * total[n + pairs]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    double u = 0.0;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) u += red[i];
    *loss = (float)(u / pairs);
  }
}

constexpr int MAX_BLOCKS = 148 * 16;

template <typename T, int MODE, int TPR, int NV, int THREADS>
int run_forward(const RowArgs& a, int* count, float* logp, float2* lse, float* slope, void* dlogits, double* partial, double* ratio, int* blocks,
                cudaStream_t stream) {
  const long long need = ((long long)a.rows + THREADS / TPR - 1) / (THREADS / TPR);
  // Warps that read a row ahead start once (178 us for 184, 110080 rows of 2024 with the gradient); else short blocks even out the hidden
  // rows' share (92 us for 106, 1016 rows of 151936).
  const long long fit = (long long)sb_num_sms() * (TPR == 32 && MODE == LOSS_POLICY ? resident_warps<MODE, TPR>() * 32 : 2048) / THREADS;
  const long long cap = fit < MAX_BLOCKS ? fit : MAX_BLOCKS;
  *blocks = (int)(need < cap ? need : cap);
  if (MODE == LOSS_POLICY && (!a.mask || a.rows / a.C <= COUNT_LIMIT))
    rows_forward_kernel<T, MODE, TPR, NV, THREADS, MODE == LOSS_POLICY><<<*blocks, THREADS, 0, stream>>>(a, count, logp, lse, slope, dlogits, partial, ratio);
  else
    rows_forward_kernel<T, MODE, TPR, NV, THREADS, false><<<*blocks, THREADS, 0, stream>>>(a, count, logp, lse, slope, dlogits, partial, ratio);
  return (int)cudaGetLastError();
}

template <typename T, int MODE>
int forward(const RowArgs& a, int* count, float* logp, float2* lse, float* slope, void* dlogits, double* partial, double* ratio, int* blocks,
            cudaStream_t stream) {
  // a row that fits eight 16-byte groups per thread of a warp or block stays in registers; a thread's groups beyond the row cost as much
  // as those within it
  const long long groups = a.V / Vec<T>::N;
  if (groups <= 32 * 2) return run_forward<T, MODE, 32, 2, 256>(a, count, logp, lse, slope, dlogits, partial, ratio, blocks, stream);
  if (groups <= 32 * 4) return run_forward<T, MODE, 32, 4, 128>(a, count, logp, lse, slope, dlogits, partial, ratio, blocks, stream);
  if (groups <= 32 * 8) return run_forward<T, MODE, 32, 8, 128>(a, count, logp, lse, slope, dlogits, partial, ratio, blocks, stream);
  if (groups <= 128 * 4) return run_forward<T, MODE, 128, 4, 128>(a, count, logp, lse, slope, dlogits, partial, ratio, blocks, stream);
  if (groups <= 128 * 8) return run_forward<T, MODE, 128, 8, 128>(a, count, logp, lse, slope, dlogits, partial, ratio, blocks, stream);
  if (groups <= 512 * 4) return run_forward<T, MODE, 512, 4, 512>(a, count, logp, lse, slope, dlogits, partial, ratio, blocks, stream);
  if (groups <= 512 * 8) return run_forward<T, MODE, 512, 8, 512>(a, count, logp, lse, slope, dlogits, partial, ratio, blocks, stream);
  return run_forward<T, MODE, 256, 0, 256>(a, count, logp, lse, slope, dlogits, partial, ratio, blocks, stream);
}

template <typename T>
int gradient(const RowArgs& a, const float2* lse, const float* slope, const float* seq_slope, const float* upstream, int unless_one, void* dlogits,
             cudaStream_t stream) {
  const long long cap = (long long)sb_num_sms() * 8;
  const long long groups = a.V / Vec<T>::N, by8 = ((long long)a.rows + 7) / 8;
  const int warps = (int)(by8 < cap ? by8 : cap), whole = (int)(a.rows < cap ? a.rows : cap);
  if (groups <= 32 * 2) rows_grad_kernel<T, 32, 2, 256><<<warps, 256, 0, stream>>>(a, lse, slope, seq_slope, upstream, unless_one, dlogits);
  else if (groups <= 32 * 8) rows_grad_kernel<T, 32, 8, 256><<<warps, 256, 0, stream>>>(a, lse, slope, seq_slope, upstream, unless_one, dlogits);
  else rows_grad_kernel<T, 256, 8, 256><<<whole, 256, 0, stream>>>(a, lse, slope, seq_slope, upstream, unless_one, dlogits);
  return (int)cudaGetLastError();
}

bool fill(RowArgs& a, const void* logits, long long sn, long long st, long long sc, const long long* targets, const uint8_t* mask, long long N, int T, int C,
          int V) {
  if (!logits || !targets || N <= 0 || T <= 0 || C <= 0 || V <= 0) return false;
  a = RowArgs{};
  a.logits = logits; a.sn = sn; a.st = st; a.sc = sc;
  a.targets = targets; a.mask = mask;
  if (N * T * C >= (1ll << 31) - (1 << 20)) return false;       // rows, and a grid's step beyond them, are counted in 32 bits
  a.rows = (int)(N * T * C);
  a.T = T; a.C = C; a.V = V;
  a.by_c = divisor(C); a.by_t = divisor(T);
  return true;
}

}  // namespace

// Logit types: 0 = bf16, 1 = fp16, 2 = fp32.  `partial`: at least sb_sequence_loss_blocks() doubles.
SB_API int sb_sequence_loss_blocks() { return MAX_BLOCKS; }

SB_API int sb_policy_loss_fwd(const void* logits, int type, long long sn, long long st, long long sc, const long long* targets, const uint8_t* mask,
                              const float* old_logp, const float* ref_logp, const float* adv, long long N, int T, int C, int V, float clip_lo,
                              float clip_hi, float kl_beta, int* count, double* partial, float* loss, float* logp, float2* lse, float* slope,
                              void* dlogits, cudaStream_t stream) {
  RowArgs a;
  if (!fill(a, logits, sn, st, sc, targets, mask, N, T, C, V) || !old_logp || !adv || !count || !partial || !loss || !logp || !lse || !slope)
    return SB_BAD_ARGUMENT;
  a.old = old_logp; a.ref = ref_logp; a.adv = adv;
  a.clip_lo = clip_lo; a.clip_hi = clip_hi; a.kl_beta = kl_beta;
  a.log_lo = clip_lo < 1.f ? log(1.0 - (double)clip_lo) : -HUGE_VAL;
  a.log_hi = log(1.0 + (double)clip_hi);
  if (mask && N * T > COUNT_LIMIT) count_kernel<<<1, 1024, 0, stream>>>(mask, a.rows, C, count);
  int blocks = 0, rc;
  if (type == 0) rc = forward<__nv_bfloat16, LOSS_POLICY>(a, count, logp, lse, slope, dlogits, partial, nullptr, &blocks, stream);
  else if (type == 1) rc = forward<__half, LOSS_POLICY>(a, count, logp, lse, slope, dlogits, partial, nullptr, &blocks, stream);
  else if (type == 2) rc = forward<float, LOSS_POLICY>(a, count, logp, lse, slope, dlogits, partial, nullptr, &blocks, stream);
  else return SB_BAD_ARGUMENT;
  if (rc) return rc;
  policy_finish_kernel<<<1, 1024, 0, stream>>>(partial, blocks, count, loss);
  return (int)cudaGetLastError();
}

SB_API int sb_preference_loss_fwd(const void* logits, int type, long long sn, long long st, long long sc, const long long* targets, const uint8_t* mask,
                                  const float* ref_logp, long long N, int T, int C, int V, int kind, float beta, const float* gap, double* ratio,
                                  double* total, float* loss, float* rewards, float* seq_slope, float2* lse, cudaStream_t stream) {
  RowArgs a;
  if (!fill(a, logits, sn, st, sc, targets, mask, N, T, C, V) || (N & 1) || N > (1 << 30) || !ref_logp || !ratio || !total || !loss || !rewards || !seq_slope ||
      !lse || kind < 0 || kind > 2 || (kind == 2 && !gap))
    return SB_BAD_ARGUMENT;
  a.ref = ref_logp;
  int blocks = 0, rc;
  if (type == 0) rc = forward<__nv_bfloat16, LOSS_PREFERENCE>(a, nullptr, nullptr, lse, nullptr, nullptr, nullptr, ratio, &blocks, stream);
  else if (type == 1) rc = forward<__half, LOSS_PREFERENCE>(a, nullptr, nullptr, lse, nullptr, nullptr, nullptr, ratio, &blocks, stream);
  else if (type == 2) rc = forward<float, LOSS_PREFERENCE>(a, nullptr, nullptr, lse, nullptr, nullptr, nullptr, ratio, &blocks, stream);
  else return SB_BAD_ARGUMENT;
  if (rc) return rc;
  const bool one = a.rows <= ONE_BLOCK_ROWS;
  if (!one) {
    ratio_kernel<<<(int)N, 256, 0, stream>>>(ratio, (long long)T * C, total);
    rc = (int)cudaGetLastError();
    if (rc) return rc;
  }
  preference_finish_kernel<<<1, one ? 1024 : 256, 0, stream>>>(one ? ratio : nullptr, (long long)T * C, total, (int)(N / 2), kind, beta, gap, loss, rewards, seq_slope);
  return (int)cudaGetLastError();
}

SB_API int sb_sequence_loss_bwd(const void* logits, int type, long long sn, long long st, long long sc, const long long* targets, const uint8_t* mask,
                                long long N, int T, int C, int V, const float2* lse, const float* slope, const float* seq_slope, const float* upstream,
                                int unless_one, void* dlogits, cudaStream_t stream) {
  RowArgs a;
  if (!fill(a, logits, sn, st, sc, targets, mask, N, T, C, V) || !lse || (!slope && !seq_slope) || !upstream || !dlogits) return SB_BAD_ARGUMENT;
  if (type == 0) return gradient<__nv_bfloat16>(a, lse, slope, seq_slope, upstream, unless_one, dlogits, stream);
  if (type == 1) return gradient<__half>(a, lse, slope, seq_slope, upstream, unless_one, dlogits, stream);
  if (type == 2) return gradient<float>(a, lse, slope, seq_slope, upstream, unless_one, dlogits, stream);
  return SB_BAD_ARGUMENT;
}
