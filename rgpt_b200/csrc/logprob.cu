// Log-probabilities of labels under rows of logits, and the two post-training losses built on them.
//
//   token_logprobs      lse = log sum_j e^{x_j}, logp = x_label - lse, and its backward
//                       dx_j = g ([j = label] - e^{x_j - lse})
//   preference_loss     pairs (chosen p, rejected p + P) of sequences with summed (or mean) log-probabilities s:
//                       h = beta ((s_c - s_r) - (ref_c - ref_r)) - margin, a loss of h, and the rows' gradients
//   policy_loss         clipped policy ratio with a KL term, per token, and the rows' gradients
//
// Logits are bf16, fp16 or fp32, row (b, t) at b * sb + t * st elements, unit stride along the vocabulary, any
// alignment. A token is scored when its label lies in [0, V) and is not ignore_index; an unscored row is not
// read, has log-probability 0 and a zero gradient. All statistics are fp32 or wider: maxima exact, sums of
// exponentials fp32 per thread, lse = max + log(sum) and the label's log-probability in fp64 (one rounding to
// fp32 when stored), sums over a sequence and over the batch in fp64 in a fixed order.
//
// A row of the type's lowest values is uniform. A row without a finite logit, or with +inf or NaN, gives NaN, as
// log(softmax) does.
#include <cuda_fp16.h>

#include "common.cuh"
#include "rgpt.h"

namespace rgpt {

constexpr float LP_LOG2E = 1.4426950408889634f;
constexpr double LP_EX2_MEAN = -5.25e-8;  // of ex2.approx.ftz.f32 over [-16, 0], measured on sm_100a
constexpr float LP_LOG2E_LO = (float)(1.4426950408889634 - (double)LP_LOG2E);  // what fp32 leaves of it, 1.9e-8
constexpr int LP_THREADS = 256;
// A stored lse carries 2^-24 |lse| of rounding into every probability of the backward: 4e-6 at this size, less than a
// sum of exponentials has of its own. Rows beyond it (a row of the type's lowest values, say) are summed again.
constexpr float LP_LSE_EXACT = 64.0f;
constexpr float LP_LOW = -2e38f;  // c * x is finite above it
constexpr float LP_WIDE = 1048576.0f;

// A [B, T] grid of rows over a strided tensor.
struct LpRows {
  long long sb, st;
  int T;
  __device__ __forceinline__ unsigned batch(long long row) const { return (unsigned)row / (unsigned)T; }  // rows < 2^31
  __device__ __forceinline__ long long offset(long long row) const {
    const unsigned b = batch(row);
    return (long long)b * sb + (long long)((unsigned)row - b * (unsigned)T) * st;
  }
};

// A pair of floats in one 64-bit register: the packed instructions take and give it as it is.
typedef unsigned long long F2;
__device__ __forceinline__ F2 f2(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 f2_get(F2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
  F2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) {
  F2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) {
  F2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ F2 f2_ex2(F2 t) {
  const float2 v = f2_get(t);
  return f2(ex2_approx(v.x), ex2_approx(v.y));
}

template <typename E>
struct LpType;
template <>
struct LpType<__nv_bfloat16> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16(v); }
  static constexpr uint32_t LOWEST = 0xFF80FF80u;  // -inf, twice
  static __device__ __forceinline__ void unpack(const uint4& u, F2 (&f)[4]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = f2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xFFFF0000u));
  }
  static __device__ __forceinline__ float max8(const uint4& u) {  // packed compares: exact
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    const float2 m = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(m.x, m.y);
  }
  static __device__ __forceinline__ uint4 pack(const F2 (&f)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 p = f2_get(f[k]);
      w[k] = pack_bf16x2(p.x, p.y);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct LpType<__half> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
  static constexpr uint32_t LOWEST = 0xFC00FC00u;
  static __device__ __forceinline__ void unpack(const uint4& u, F2 (&f)[4]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      f[k] = f2(p.x, p.y);
    }
  }
  static __device__ __forceinline__ float max8(const uint4& u) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
    const float2 m = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(m.x, m.y);
  }
  static __device__ __forceinline__ uint4 pack(const F2 (&f)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 p = f2_get(f[k]);
      const __half2 h = __floats2half2_rn(p.x, p.y);
      w[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct LpType<float> {
  static constexpr int VEC = 4;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
  static constexpr uint32_t LOWEST = 0xFF800000u;
  static __device__ __forceinline__ void unpack(const uint4& u, F2 (&f)[2]) {
    f[0] = f2(__uint_as_float(u.x), __uint_as_float(u.y));
    f[1] = f2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
  static __device__ __forceinline__ float max8(const uint4& u) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  static __device__ __forceinline__ uint4 pack(const F2 (&f)[2]) {
    const float2 p = f2_get(f[0]), q = f2_get(f[1]);
    return make_uint4(__float_as_uint(p.x), __float_as_uint(p.y), __float_as_uint(q.x), __float_as_uint(q.y));
  }
};

__device__ __forceinline__ bool lp_scored(long long label, long long ignore_index, int V) {
  return label != ignore_index && label >= 0 && label < V;
}

// The reference point of an exponent: -inf (nothing seen yet) is replaced by 0, so that e^{-inf - 0} = 0.
__device__ __forceinline__ float lp_ref(float m) { return m == -INFINITY ? 0.f : m; }

// A running (M, sum of 2^{c x - M}) in base 2, c = log2 e in two parts: two fused multiply-adds and one exponential an
// element. What is the same for every row would add up over a long sequence, so it is kept small: c's first part alone
// makes log-probabilities some 6e-8 too high; M = ceil(c max) is a whole number, so that rescaling a sum is exact (with
// any other M the hardware exponential's mean relative error, -5.25e-8 over a binade, comes in at each rescaling: 2e-7
// in all); and that error of the elements themselves is taken off the row's sum at the end. Elements up to LP_LOW, where c x
// overflows, count as nothing (M = -inf). A row that holds nothing else, or whose |M| is so large that c max - M may be
// (beyond LP_WIDE its 2^-24 |M| is no longer small), takes the careful pass: e^{x - max} after the subtraction.
struct LpSum {
  float m = -INFINITY, s = 0.f;
  __device__ __forceinline__ void merge(float om, float os) {
    const float nm = fmaxf(m, om), r = lp_ref(nm);
    s = s * ex2_approx(m - r) + os * ex2_approx(om - r);
    m = nm;
  }
  // U vectors at once: one rescaling of the sum for all of them
  template <typename L, int U>
  __device__ __forceinline__ void add(const uint4 (&u)[U]) {
    float lm = L::max8(u[0]);
#pragma unroll
    for (int k = 1; k < U; ++k) lm = fmaxf(lm, L::max8(u[k]));
    const float nm = fmaxf(m, lm > LP_LOW ? ceilf(lm * LP_LOG2E) : -INFINITY), r = lp_ref(nm);
    s *= ex2_approx(m - r);
    m = nm;
    const F2 nr = f2(-r, -r), l2e = f2(LP_LOG2E, LP_LOG2E), lo = f2(LP_LOG2E_LO, LP_LOG2E_LO);
    F2 a0 = f2(s, 0.f), a1 = f2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < U; ++k) {
      F2 f[L::VEC / 2];
      L::unpack(u[k], f);
#pragma unroll
      for (int j = 0; j < L::VEC / 2; j += 2) {
        a0 = f2_add(a0, f2_ex2(f2_fma(f[j], lo, f2_fma(f[j], l2e, nr))));
        a1 = f2_add(a1, f2_ex2(f2_fma(f[j + 1], lo, f2_fma(f[j + 1], l2e, nr))));
      }
    }
    const float2 b = f2_get(f2_add(a0, a1));
    s = b.x + b.y;
  }
  __device__ __forceinline__ void add(float f) {
    const float nm = fmaxf(m, f > LP_LOW ? ceilf(f * LP_LOG2E) : -INFINITY), r = lp_ref(nm);
    s = s * ex2_approx(m - r) + ex2_approx(fmaf(f, LP_LOG2E_LO, fmaf(f, LP_LOG2E, -r)));
    m = nm;
  }
};

// What a row's sum comes to: probabilities e^{x - lse} = 2^{c (x - a) - b} * inv. The subtraction comes first, so that
// what fp32 leaves of c and of the product goes with x - a and not with x (2^{c x - M} / sum, in one fused operation an
// element, makes every probability of a row of logits near 1000 some 1e-5 too small). After the plain pass a is lse
// rounded to fp32 and b the rest of it in base 2, after a careful pass a = max and b = 0.
struct LpRow {
  float a, b, inv;
  double lse;
};

// Elements of a row before its first 16-byte boundary.
template <typename E>
__device__ __forceinline__ int lp_head(const E* x, int V) {
  const int h = (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(E));
  return h < V ? h : V;
}

// Who works on a row: one CTA; the CTAs of a cluster, when there are too few rows for the SMs; or one warp, when rows
// are short. CTA `part` of a cluster takes its share of the row's 16-byte vectors and of the elements outside them.
enum LpTeam { LP_CTA = 0, LP_CLUSTER = 1, LP_WARP = 2 };
struct LpShare {
  int part, parts;
  __device__ __forceinline__ int lo(int n) const { return (int)((long long)n * part / parts); }
  __device__ __forceinline__ int hi(int n) const { return (int)((long long)n * (part + 1) / parts); }
};
template <int W>
__device__ __forceinline__ LpShare lp_share() {
  LpShare s = {0, 1};
  if constexpr (W == LP_CLUSTER) {
    s.part = (int)cluster_ctarank();
    s.parts = (int)cluster_nctarank();
  }
  return s;
}
template <int W>
__device__ __forceinline__ int lp_rank() {  // of this thread among those of its CTA that share its row
  return W == LP_WARP ? (int)(threadIdx.x & 31) : (int)threadIdx.x;
}
template <int W>
constexpr int lp_size(int cta_threads) {
  return W == LP_WARP ? 32 : cta_threads;
}
template <int W>
__device__ __forceinline__ long long lp_row(LpShare sh) {
  if (W == LP_WARP) return (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  return (long long)(blockIdx.x / sh.parts);
}

// LP_UNROLL vectors in flight a thread: 4 x 16 bytes x 1280 threads on an SM cover HBM's latency at its full rate.
constexpr int LP_UNROLL = 4;

// One (m, s) for the row from each thread's, by MERGE: the same in every thread of every CTA of the row, and on return
// all of them have read it.
template <int W, typename MERGE>
__device__ __forceinline__ float2 lp_join(float2 a, LpShare sh, MERGE&& merge) {
  __shared__ float2 sm[LP_THREADS / 32];
  __shared__ float2 all;
  for (int o = 16; o > 0; o >>= 1)
    a = merge(a, make_float2(__shfl_xor_sync(0xffffffffu, a.x, o), __shfl_xor_sync(0xffffffffu, a.y, o)));
  if constexpr (W == LP_WARP)  // which of two sums is scaled first rounds differently: lane 0's, for every lane
    return make_float2(__shfl_sync(0xffffffffu, a.x, 0), __shfl_sync(0xffffffffu, a.y, 0));
  __syncthreads();  // an earlier join may still be read
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = a;
  __syncthreads();
  float2 r = sm[0];
#pragma unroll
  for (int w = 1; w < LP_THREADS / 32; ++w)
    if (w < (int)(blockDim.x >> 5)) r = merge(r, sm[w]);
  if constexpr (W == LP_CLUSTER) {
    if (threadIdx.x == 0) all = r;
    cluster_sync_all();
    r = ld_shared_cluster_f2(mapa_shared(smem_u32(&all), 0));
    for (int c = 1; c < sh.parts; ++c) r = merge(r, ld_shared_cluster_f2(mapa_shared(smem_u32(&all), (uint32_t)c)));
    cluster_sync_all();  // no CTA leaves, or writes `all` again, while another still reads it
  }
  return r;
}

// M ln2 + log(s) for a normal s: log(s) from the mantissa in [0.75, 1.5) in fp32 (absolute error 2^-25) and the exponent
// in fp64
__device__ __forceinline__ double lp_log(double M, float s) {
  constexpr double LN2 = 0.69314718055994530942;
  const int e = (int)((__float_as_uint(s) - 0x3F400000u) & 0xFF800000u) >> 23;
  const float f = __uint_as_float(__float_as_uint(s) - ((uint32_t)e << 23));
  return fma(M + (double)e, LN2, (double)logf(f));
}
// The finished row from its joined (M, s).
__device__ __forceinline__ LpRow lp_finish(float2 r) {
  const double lse = lp_log((double)r.x, r.y) - LP_EX2_MEAN;
  const float a = (float)lse;
  return LpRow{a, (float)((lse - (double)a) * 1.4426950408889634), 1.f, lse};
}
// The label's log-probability; rounding may not make a sure label more than sure.
__device__ __forceinline__ double lp_label(float xl, const LpRow& r) {
  const double lp = (double)xl - r.lse;
  return lp > 0.0 ? 0.0 : lp;
}
__device__ __forceinline__ bool lp_plain(float2 r) {
  return fabsf(r.x) <= LP_WIDE && r.y < INFINITY;  // a NaN in the row makes the sum NaN
}

// The careful pass over a row in global memory by n threads (index t), joined by `join` (the same in all of them).
template <typename E, typename J>
__device__ __noinline__ LpRow lp_careful(const E* x, int V, int t, int n, J join) {
  float top = -INFINITY, sum = 0.f;
#pragma unroll 1
  for (int j = t; j < V; j += n) top = fmaxf(top, LpType<E>::get(x[j]));
  const float ref = lp_ref(join(make_float2(top, 0.f), true).x);
#pragma unroll 1
  for (int j = t; j < V; j += n) sum += ex2_approx((LpType<E>::get(x[j]) - ref) * LP_LOG2E);
  sum = join(make_float2(sum, 0.f), false).x;
  // a sum of 0 (nothing but -inf) gives -inf, an infinite or NaN one itself
  const double l = sum > 0.f && sum < INFINITY ? lp_log(0.0, sum) : sum == 0.f ? -INFINITY : (double)sum;
  return LpRow{ref, 0.f, 1.f / sum, (double)ref + l};
}
__device__ __forceinline__ float2 lp_merge(float2 p, float2 q) {
  LpSum t;
  t.m = p.x, t.s = p.y;
  t.merge(q.x, q.y);
  return make_float2(t.m, t.s);
}
template <int W>
struct LpTeamJoin {
  LpShare sh;
  __device__ float2 operator()(float2 v, bool max) const {
    return max ? lp_join<W>(v, sh, [](float2 p, float2 q) { return make_float2(fmaxf(p.x, q.x), 0.f); })
               : lp_join<W>(v, sh, [](float2 p, float2 q) { return make_float2(p.x + q.x, 0.f); });
  }
};
// The careful pass by a row's whole team.
template <typename E, int W, int THREADS>
__device__ __forceinline__ LpRow lp_team_careful(const E* x, int V, LpShare sh) {
  constexpr int N = lp_size<W>(THREADS);
  return lp_careful(x, V, sh.part * N + lp_rank<W>(), sh.parts * N, LpTeamJoin<W>{sh});
}

// The sum of one short row, the same in every thread of its CTA or warp, all of which have read it on return.
template <typename E, int W>
__device__ __forceinline__ LpRow lp_row_sum(const E* x, int V) {
  using L = LpType<E>;
  constexpr int N = lp_size<W>(LP_THREADS);
  const LpShare sh = {0, 1};
  const int head = lp_head(x, V), nvec = (V - head) / L::VEC;
  LpSum a;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  const int wend = nvec + (int)(threadIdx.x & 31);  // the loops are uniform over a warp
  auto add = [&](auto unroll, int v) {
    constexpr int U = decltype(unroll)::value;
    uint4 u[U];
#pragma unroll
    for (int k = 0; k < U; ++k)
      u[k] = v + k * N < nvec ? xv[v + k * N] : make_uint4(L::LOWEST, L::LOWEST, L::LOWEST, L::LOWEST);
    a.template add<L, U>(u);
  };
  int v = lp_rank<W>();
  for (; v + N < wend; v += LP_UNROLL * N) {
    if (v + 2 * N < wend) add(std::integral_constant<int, LP_UNROLL>{}, v);
    else add(std::integral_constant<int, 2>{}, v);
  }
  if (v < wend) add(std::integral_constant<int, 1>{}, v);
  const int rest = V - nvec * L::VEC;  // the head, then the tail behind the vectors
  for (int j = lp_rank<W>(); j < rest; j += N) a.add(L::get(x[j < head ? j : j + nvec * L::VEC]));
  const float2 r = lp_join<W>(make_float2(a.m, a.s), sh, lp_merge);
  if (lp_plain(r)) return lp_finish(r);
  return lp_team_careful<E, W, LP_THREADS>(x, V, sh);
}

// 2^{c (x - a) - b} of two logits, times a factor
struct LpProb {
  F2 na, nb, k;
  __device__ __forceinline__ LpProb(float a, float b, float factor)
      : na(f2(-a, -a)), nb(f2(-b, -b)), k(f2(factor, factor)) {}
  __device__ __forceinline__ F2 operator()(F2 f) const {
    return f2_mul(f2_ex2(f2_fma(f2_add(f, na), f2(LP_LOG2E, LP_LOG2E), nb)), k);
  }
  __device__ __forceinline__ float one(float f) const { return f2_get((*this)(f2(f, 0.f))).x; }
};
// adds coef to element `at` of a vector
template <typename L>
__device__ __forceinline__ void lp_at_label(F2 (&f)[L::VEC / 2], int at, float coef) {
#pragma unroll
  for (int k = 0; k < L::VEC / 2; ++k) f[k] = f2_add(f[k], f2(2 * k == at ? coef : 0.f, 2 * k + 1 == at ? coef : 0.f));
}

// A vector of the gradient; the label is its element `at`.
template <typename E>
__device__ __forceinline__ uint4 lp_grad_vec(const uint4& u, int at, float coef, const LpProb& prob) {
  using L = LpType<E>;
  F2 f[L::VEC / 2];
  L::unpack(u, f);
#pragma unroll
  for (int k = 0; k < L::VEC / 2; ++k) f[k] = prob(f[k]);
  if (at >= 0 && at < L::VEC) lp_at_label<L>(f, at, coef);
  return L::pack(f);
}
// Its elements i = from, from + step .. of those outside the vectors: `head` before them, then the ones behind.
template <typename E>
__device__ __forceinline__ void lp_write_rest(const E* x, E* d, int label, float coef, int head, int vec_elems, int from,
                                              int to, int step, const LpProb& prob) {
  using L = LpType<E>;
  for (int i = from; i < to; i += step) {
    const int j = i < head ? i : i + vec_elems;
    const float g = prob.one(L::get(x[j]));
    d[j] = L::put(j == label ? g + coef : g);
  }
}
// 16 bytes at an address of the type's alignment only: by 4-byte words, two bytes on where that address lies inside one (a
// word is never split between what may be read and what may not).
__device__ __forceinline__ uint4 lp_load_any(const float* p) {
  return make_uint4(__float_as_uint(p[0]), __float_as_uint(p[1]), __float_as_uint(p[2]), __float_as_uint(p[3]));
}
template <typename E>
__device__ __forceinline__ uint4 lp_load_any(const E* p) {
  static_assert(sizeof(E) == 2, "16-bit types");
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  const uint32_t* w = reinterpret_cast<const uint32_t*>(at & ~(uintptr_t)3);
  const uint32_t a = w[0], b = w[1], c = w[2], d = w[3];
  if ((at & 2) == 0) return make_uint4(a, b, c, d);
  const uint32_t e = w[4];
  return make_uint4(__funnelshift_r(a, b, 16), __funnelshift_r(b, c, 16), __funnelshift_r(c, d, 16),
                    __funnelshift_r(d, e, 16));
}
template <typename E>
__device__ __forceinline__ bool lp_aligned(const E* x, const E* d) {
  return ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
}

// This CTA's share of coef * ([j = label] - p(x_j)) over one row; prob gives -coef * p. d may be x: each thread reads
// an element before it writes the same one. LAST: nobody reads the row after this, so its lines may leave L2 first.
template <typename E, int W, bool LAST>
__device__ __forceinline__ void lp_write_grad(const E* x, E* d, int V, int label, float coef, LpShare sh,
                                              const LpProb& prob) {
  using L = LpType<E>;
  constexpr int N = lp_size<W>(LP_THREADS);
  const bool same = lp_aligned(x, d);
  const int head = lp_head(d, V), nvec = (V - head) / L::VEC;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  uint4* dv = reinterpret_cast<uint4*>(d + head);
  auto one = [&](const uint4& u, int at) { return lp_grad_vec<E>(u, at, coef, prob); };
  int v = sh.lo(nvec) + lp_rank<W>();
  const int vend = sh.hi(nvec);
  if (!same) {  // stores by vectors, loads by what x's alignment allows (4096 rows of 50257 bf16: 198 us; aligned 137)
#pragma unroll 1
    for (; v < vend; v += N) __stcs(&dv[v], one(lp_load_any(x + head + (long long)v * L::VEC), label - head - v * L::VEC));
  }
  if constexpr (W == LP_WARP) {  // short rows: one step takes most of them, its last vectors from some lanes only
    for (; v - lp_rank<W>() < vend; v += LP_UNROLL * N) {
      uint4 u[LP_UNROLL];
#pragma unroll
      for (int k = 0; k < LP_UNROLL; ++k)
        if (v + k * N < vend) u[k] = xv[v + k * N];
#pragma unroll
      for (int k = 0; k < LP_UNROLL; ++k)
        if (v + k * N < vend) __stcs(&dv[v + k * N], one(u[k], label - head - (v + k * N) * L::VEC));
    }
  }
  for (; v + (LP_UNROLL - 1) * N < vend; v += LP_UNROLL * N) {
    uint4 u[LP_UNROLL];
#pragma unroll
    for (int k = 0; k < LP_UNROLL; ++k) u[k] = LAST ? __ldcs(&xv[v + k * N]) : xv[v + k * N];
#pragma unroll
    for (int k = 0; k < LP_UNROLL; ++k)
      __stcs(&dv[v + k * N], one(u[k], label - head - (v + k * N) * L::VEC));  // not kept in L2
  }
  for (; v < vend; v += N) dv[v] = one(xv[v], label - head - v * L::VEC);
  const int rest = V - nvec * L::VEC;
  lp_write_rest<E>(x, d, label, coef, head, nvec * L::VEC, sh.lo(rest) + lp_rank<W>(), sh.hi(rest), N, prob);
}

template <typename E, int W>
__device__ __forceinline__ void lp_write_zero(E* d, int V, LpShare sh) {
  using L = LpType<E>;
  const int head = lp_head(d, V), nvec = (V - head) / L::VEC;
  uint4* dv = reinterpret_cast<uint4*>(d + head);
  for (int v = sh.lo(nvec) + lp_rank<W>(); v < sh.hi(nvec); v += lp_size<W>(blockDim.x))
    __stcs(&dv[v], make_uint4(0u, 0u, 0u, 0u));
  const int rest = V - nvec * L::VEC;
  for (int i = sh.lo(rest) + lp_rank<W>(); i < sh.hi(rest); i += lp_size<W>(blockDim.x))
    d[i < head ? i : i + nvec * L::VEC] = L::put(0.f);
}

// ---------------------------------------------------------------------------- rows through shared memory
// This CTA's share of a row's vectors, brought in by bulk copies of VECS each, in order, into `slots` places that are
// used again once every thread is done with them. Waits are bounded: after one has run out (the device error word says
// so) nothing more is issued or waited for, but for what is still on its way at the end.
template <int VECS>
struct LpStage {
  const uint4* src;
  uint4* place;
  uint64_t* full;
  int n, pieces, slots, issued;
  bool ok;
  bool passing;  // its lines may leave L2 first
  const uint64_t policy;
  __device__ __forceinline__ LpStage(const uint4* src_, int n_, void* smem, uint64_t* full_, int slots_, bool passing_)
      : src(src_), place(reinterpret_cast<uint4*>(smem)), full(full_), n(n_), pieces((n_ + VECS - 1) / VECS),
        slots(slots_), issued(0), ok(true), passing(passing_), policy(l2_evict_first()) {}
  __device__ __forceinline__ int size(int c) const { return min(VECS, n - c * VECS); }
  __device__ __forceinline__ void issue(int c) {  // thread 0
    const uint32_t bytes = 16u * (uint32_t)size(c);
    mbar_arrive_expect_tx(&full[c % slots], bytes);
    uint4* at = place + (c % slots) * VECS;
    if (passing) bulk_load_1d(at, src + (long long)c * VECS, bytes, &full[c % slots], policy);
    else bulk_load_1d(at, src + (long long)c * VECS, bytes, &full[c % slots]);
    issued = c + 1;
  }
  // all threads, first
  __device__ __forceinline__ void start() {
    if (threadIdx.x == 0) {
      for (int i = 0; i < min(pieces, slots); ++i) mbar_init(&full[i], 1);
      fence_barrier_init();
      for (int i = 0; i < min(pieces, slots); ++i) issue(i);
    }
    __syncthreads();
  }
  __device__ __forceinline__ const uint4* wait(int c) {
    if (ok && !mbar_wait(&full[c % slots], (uint32_t)(c / slots) & 1u, nullptr)) {
      ok = false;
      if (threadIdx.x == 0)  // the copies on their way must land before the CTA's shared memory is given up
        for (int i = c; i < issued; ++i) mbar_wait(&full[i % slots], (uint32_t)(i / slots) & 1u, nullptr);
    }
    return place + (c % slots) * VECS;
  }
  // all threads, after their reads of piece c
  __device__ __forceinline__ void next(int c) {
    if (c + slots >= pieces) return;
    __syncthreads();
    if (threadIdx.x == 0 && ok) issue(c + slots);
  }
  // A second time through, from the last piece to the first: the last ones are still in their places, the others are
  // brought in again, each into its place. Piece c comes as the place's use number (last + (last - c)) / slots, from 0,
  // where last is the place's last piece.
  __device__ __forceinline__ uint32_t back_parity(int c) const {
    const int last = pieces - 1 - (pieces - 1 - c) % slots;
    return (uint32_t)(last / slots + (last - c) / slots) & 1u;
  }
  __device__ __forceinline__ const uint4* wait_back(int c) {
    if (c < pieces - slots && ok && !mbar_wait(&full[c % slots], back_parity(c), nullptr)) {
      ok = false;
      if (threadIdx.x == 0)
        for (int i = c - 1; i > c - slots && i >= 0; --i) mbar_wait(&full[i % slots], back_parity(i), nullptr);
    }
    return place + (c % slots) * VECS;
  }
  __device__ __forceinline__ void next_back(int c) {
    if (c - slots < 0) return;
    __syncthreads();
    if (threadIdx.x == 0 && ok) issue(c - slots);
  }
};

// Adds a piece of n vectors to a thread's sum, U vectors at a time; lanes past the end of the last ones add -inf.
template <typename L, int VECS, int THREADS, int U>
__device__ __forceinline__ void lp_add_piece(LpSum& sum, const uint4* v, int n) {
  static_assert(VECS % (U * THREADS) == 0, "a whole piece takes whole steps");
  const int t = threadIdx.x;
  if (n == VECS) {
#pragma unroll 1
    for (int i = t; i < VECS; i += U * THREADS) {
      uint4 u[U];
#pragma unroll
      for (int k = 0; k < U; ++k) u[k] = v[i + k * THREADS];
      sum.template add<L, U>(u);
    }
  } else {
#pragma unroll 1
    for (int i = t; i - (t & 31) < n; i += THREADS) {  // warp-uniform
      const uint4 u[1] = {i < n ? v[i] : make_uint4(L::LOWEST, L::LOWEST, L::LOWEST, L::LOWEST)};
      sum.template add<L, 1>(u);
    }
  }
}

// The sum of one row through shared memory, the same in every thread of its CTAs, all of which have read it on return.
template <int VECS, typename E>
__device__ __forceinline__ LpStage<VECS> lp_stage(const E* x, int V, LpShare sh, void* smem, uint64_t* full, int slots,
                                                  bool passing) {
  const int head = lp_head(x, V), nvec = (V - head) / LpType<E>::VEC, lo = sh.lo(nvec);
  return LpStage<VECS>(reinterpret_cast<const uint4*>(x + head) + lo, sh.hi(nvec) - lo, smem, full, slots, passing);
}
template <typename E, int W, int THREADS, int VECS, typename F>
__device__ __forceinline__ void lp_staged_sum(LpStage<VECS>& st, const E* x, int V, LpShare sh, LpRow* out,
                                              F&& meanwhile) {
  using L = LpType<E>;
  const int head = lp_head(x, V), nvec = (V - head) / L::VEC, rest = V - nvec * L::VEC;
  st.start();
  meanwhile();
  LpSum a;
  for (int j = sh.lo(rest) + threadIdx.x; j < sh.hi(rest); j += THREADS)
    a.add(L::get(x[j < head ? j : j + nvec * L::VEC]));
  for (int c = 0; c < st.pieces; ++c) {
    lp_add_piece<L, VECS, THREADS, 4>(a, st.wait(c), st.size(c));
    st.next(c);
  }
  const float2 q = lp_join<W>(make_float2(a.m, a.s), sh, lp_merge);
  *out = lp_plain(q) ? lp_finish(q) : lp_team_careful<E, W, THREADS>(x, V, sh);
}

// lp_write_grad by the threads and from the stage of lp_staged_sum, for d of x's alignment (mod 16).
template <typename E, int THREADS, int VECS>
__device__ __forceinline__ void lp_staged_grad(LpStage<VECS>& st, const E* x, E* d, int V, int label, float coef,
                                               LpShare sh, const LpProb& prob) {
  using L = LpType<E>;
  constexpr int U = 4;
  static_assert(VECS % (U * THREADS) == 0, "a whole piece takes whole steps");
  const int head = lp_head(x, V), nvec = (V - head) / L::VEC, rest = V - nvec * L::VEC, lo = sh.lo(nvec);
  uint4* dv = reinterpret_cast<uint4*>(d + head) + lo;
  st.passing = true;  // nobody reads the row after this
  for (int c = st.pieces - 1; c >= 0; --c) {
    const uint4* v = st.wait_back(c);
    const int n = st.size(c), first = c * VECS;
    auto one = [&](uint4 u, int i) {
      __stcs(&dv[first + i], lp_grad_vec<E>(u, label - head - (lo + first + i) * L::VEC, coef, prob));
    };
    if (n == VECS) {
#pragma unroll 1
      for (int i = threadIdx.x; i < VECS; i += U * THREADS) {
        uint4 u[U];
#pragma unroll
        for (int k = 0; k < U; ++k) u[k] = v[i + k * THREADS];
#pragma unroll
        for (int k = 0; k < U; ++k) one(u[k], i + k * THREADS);
      }
    } else {
#pragma unroll 1
      for (int i = threadIdx.x; i < n; i += THREADS) one(v[i], i);
    }
    st.next_back(c);
  }
  lp_write_rest<E>(x, d, label, coef, head, nvec * L::VEC, sh.lo(rest) + (int)threadIdx.x, sh.hi(rest), THREADS, prob);
}

// ---------------------------------------------------------------------------- token log-probabilities
// Forward for long rows: one CTA a row (or a share of it), 16 KB of it in flight; nine small CTAs an SM, each in its own
// phase, keep the copies and the exponentials going at the same time (4092 rows of 50304 bf16 logits, 2492 of them
// scored: 45 us, 5.6 TB/s; some 3 less without the exponentials; pieces of 4 KB 52; four CTAs of 256 threads an SM 7 us
// more, loads into registers 11 more). Two slots, because an SM's split into shared memory and L1 outlasts the kernel:
// with three, the backward that follows at once finds little L1 to land its loads in (forward and backward 162 us against
// 154; of 16368 rows 616 against 576).
constexpr int LP_FWD_THREADS = 128, LP_FWD_VECS = 512;
template <int W>
constexpr int LP_FWD_SLOTS = W == LP_CLUSTER ? 4 : 2;  // few rows: SMs that are not full (8 x 131072 fp32 8.4 -> 7.8 us)
// Bytes of the last rows that the forward leaves to L2's usual care, the rows before them marked to go first: with the two
// L2 halves that an SM's loads may go through, more than this does not stay (60 to 100 MB: 154 -> 150 us).
constexpr unsigned long long LP_KEEP_BYTES = 80ull << 20;
template <int W>
constexpr uint32_t LP_FWD_SMEM = LP_FWD_SLOTS<W> * LP_FWD_VECS * 16u;
template <typename E, int W>
__global__ void __launch_bounds__(LP_FWD_THREADS) logp_fwd_staged_kernel(const E* __restrict__ logits, LpRows lr, int V,
                                                                        const long long* __restrict__ labels,
                                                                        long long ignore_index,
                                                                        float* __restrict__ logps,
                                                                        float* __restrict__ lse,
                                                                        double* __restrict__ wide) {
  using L = LpType<E>;
  extern __shared__ __align__(128) uint8_t lp_smem[];
  __shared__ uint64_t full[LP_FWD_SLOTS<W>];
  griddep_wait();
  griddep_launch();
  const LpShare sh = lp_share<W>();
  const long long row = blockIdx.x / sh.parts;
  const long long label = labels[row];
  const bool first = threadIdx.x == 0 && sh.part == 0;
  if (!lp_scored(label, ignore_index, V)) {
    if (first) {
      logps[row] = 0.f;
      if (lse) lse[row] = 0.f;
      if (wide) wide[row] = 0.0;
    }
    return;
  }
  const E* x = logits + lr.offset(row);
  const float xl = first ? L::get(x[label]) : 0.f;
  LpRow r;
  // a backward begins with the last rows (see logp_bwd_kernel): those before make room for them
  const bool passing = (unsigned long long)(gridDim.x / sh.parts - 1 - row) * V * sizeof(E) > LP_KEEP_BYTES;
  auto st = lp_stage<LP_FWD_VECS>(x, V, sh, lp_smem, full, LP_FWD_SLOTS<W>, passing);
  lp_staged_sum<E, W, LP_FWD_THREADS>(st, x, V, sh, &r, [] {});
  if (first) {
    const double lp = lp_label(xl, r);
    logps[row] = (float)lp;
    if (lse) lse[row] = (float)r.lse;
    if (wide) wide[row] = lp;
  }
}

// Forward for short rows: one pass over a row with a running maximum and sum.
template <typename E, int W>
__global__ void __launch_bounds__(LP_THREADS) logp_fwd_kernel(const E* __restrict__ logits, LpRows lr, int V,
                                                              const long long* __restrict__ labels,
                                                              long long ignore_index, float* __restrict__ logps,
                                                              float* __restrict__ lse,
                                                              double* __restrict__ wide, long long M) {
  griddep_wait();
  griddep_launch();
  const long long row = lp_row<W>(LpShare{0, 1});
  if (row >= M) return;  // whole warps
  const long long label = labels[row];
  const bool first = lp_rank<W>() == 0;
  if (!lp_scored(label, ignore_index, V)) {
    if (first) {
      logps[row] = 0.f;
      if (lse) lse[row] = 0.f;
      if (wide) wide[row] = 0.0;
    }
    return;
  }
  const E* x = logits + lr.offset(row);
  const LpRow r = lp_row_sum<E, W>(x, V);
  if (first) {
    const double lp = lp_label(LpType<E>::get(x[label]), r);
    logps[row] = (float)lp;
    if (lse) lse[row] = (float)r.lse;
    if (wide) wide[row] = lp;
  }
}

// dlogits = coef * (onehot - e^{x - lse}); coef per token, or per sequence (per_seq). Elementwise, so dlogits may be
// the logits themselves.
template <typename E, int W>
__global__ void __launch_bounds__(LP_THREADS) logp_bwd_kernel(const E* logits, LpRows lr, int V,
                                                              const long long* __restrict__ labels,
                                                              long long ignore_index, const float* __restrict__ lse,
                                                              const float* __restrict__ coef, int per_seq, E* dlogits,
                                                              LpRows dr, long long M) {
  griddep_wait();
  griddep_launch();
  const LpShare sh = lp_share<W>();
  // the last rows first: the forward has left them in L2 (4092 rows of 100 KB: forward and backward 10 us less)
  const long long row = M - 1 - lp_row<W>(sh);
  if (row < 0) return;  // whole warps
  const long long label = labels[row];
  E* d = dlogits + dr.offset(row);
  if (!lp_scored(label, ignore_index, V)) {
    lp_write_zero<E, W>(d, V, sh);
    return;
  }
  const E* x = logits + lr.offset(row);
  const float l = lse[row], c = coef[per_seq ? lr.batch(row) : row];
  LpRow r = {l, 0.f, 1.f, 0.0};
  if (!(fabsf(l) <= LP_LSE_EXACT)) {
    r = lp_team_careful<E, W, LP_THREADS>(x, V, sh);
    if (W == LP_WARP) __syncwarp();  // every thread has read the row before an in-place gradient
    else __syncthreads();
  }
  lp_write_grad<E, W, false>(x, d, V, (int)label, c, sh, LpProb(r.a, r.b, -c * r.inv));
}

// ---------------------------------------------------------------------------- sums over a CTA
template <typename S>
__device__ __forceinline__ S lp_block_sum(S v, S* red) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();  // red may still be read from an earlier sum
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  S t = 0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) t += red[w];
  return t;
}

// three sums at once, in thread 0
__device__ __forceinline__ double3 lp_block_sum3(double3 v, double3* red) {
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    v.z += __shfl_xor_sync(0xffffffffu, v.z, o);
  }
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < (int)(blockDim.x >> 5); ++w) v.x += red[w].x, v.y += red[w].y, v.z += red[w].z;
  return v;
}

// ---------------------------------------------------------------------------- preference loss
struct PrefArgs {
  int kind;
  float beta, margin, smoothing, grad_scale;
  int average;
};

// loss and d loss / d h of one pair
__device__ __forceinline__ void pref_terms(const PrefArgs& a, double h, double* loss, double* dh) {
  if (a.kind == RGPT_PREF_HINGE) {
    *loss = h < 1.0 ? 1.0 - h : (h >= 1.0 ? 0.0 : h);  // NaN stays NaN
    *dh = h < 1.0 ? -1.0 : 0.0;
  } else if (a.kind == RGPT_PREF_SQUARED) {
    *loss = (h - 0.5) * (h - 0.5);
    *dh = 2.0 * (h - 0.5);
  } else {
    const double s = a.smoothing, e = exp(-fabs(h)), l = log1p(e);
    const double big = 1.0 / (1.0 + e), small = e / (1.0 + e);
    const double sig = h >= 0.0 ? big : small, sign = h >= 0.0 ? small : big;  // sigmoid(h), sigmoid(-h)
    *loss = (1.0 - s) * (fmax(-h, 0.0) + l);
    if (s > 0.0) *loss += s * (fmax(h, 0.0) + l);  // not 0 * inf
    if (isnan(h)) *loss = h;
    *dh = -(1.0 - s) * sign + s * sig;
  }
}

// A pair a warp, or for long sequences a CTA: the two sequences' log-probabilities in fp64, the margin h and the sequences'
// coefficients d loss / d (a scored token's log-probability). Where one CTA takes all pairs it writes their mean loss as
// well, which saves a launch; else a pair's loss, in fp64, takes the place of its first log-probability, which only this
// pair reads and has read.
__global__ void __launch_bounds__(256) pref_pair_kernel(double* logps,
                                                        const long long* __restrict__ labels, long long ignore_index,
                                                        int V, int P, int T, int by_warp, const float* __restrict__ ref,
                                                        PrefArgs a, float* __restrict__ seq_logps,
                                                        float* __restrict__ margins, float* __restrict__ coef,
                                                        float* __restrict__ loss_out) {
  griddep_wait();
  griddep_launch();
  __shared__ double red[8];
  const int p = by_warp ? (int)(blockIdx.x * 8 + (threadIdx.x >> 5)) : (int)blockIdx.x;
  const int step = by_warp ? 32 : 256, t0 = (int)threadIdx.x % step;
  double pair_loss = 0.0;
  if (p < P) {  // whole warps, or the whole CTA
    double s[2], n[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const long long base = (long long)(p + k * P) * T;
      double v = 0.0;
      int c = 0;
      for (int t = t0; t < T; t += step) {
        v += logps[base + t];
        if (a.average) c += lp_scored(labels[base + t], ignore_index, V) ? 1 : 0;
      }
      if (by_warp) {
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        c = __reduce_add_sync(0xffffffffu, c);
      } else {
        v = lp_block_sum(v, red);
        if (a.average) c = (int)lp_block_sum((double)c, red);
      }
      n[k] = a.average ? (double)max(c, 1) : 1.0;
      s[k] = v / n[k];
    }
    if (t0 == 0) {
      double d = s[0] - s[1];
      if (ref) d = (s[0] - (double)ref[p]) - (s[1] - (double)ref[p + P]);
      const double h = (double)a.beta * d - (double)a.margin;
      double dh;
      pref_terms(a, h, &pair_loss, &dh);
      dh *= (double)a.beta * (double)a.grad_scale / P;
      seq_logps[p] = (float)s[0];
      seq_logps[p + P] = (float)s[1];
      margins[p] = (float)h;
      coef[p] = (float)(dh / n[0]);
      coef[p + P] = (float)(-dh / n[1]);
      if (gridDim.x > 1) logps[(long long)p * T] = pair_loss;
    }
  }
  if (gridDim.x > 1) return;
  const double mean = lp_block_sum(pair_loss, red);
  if (threadIdx.x == 0) loss_out[0] = (float)(mean / P);
}

// mean of the pairs' losses, one every `step` places
__global__ void __launch_bounds__(256) pref_loss_kernel(const double* __restrict__ pair_loss, int P, long long step,
                                                        float* __restrict__ loss) {
  griddep_wait();
  griddep_launch();
  __shared__ double red[8];
  double v = 0.0;
  for (int p = threadIdx.x; p < P; p += blockDim.x) v += pair_loss[p * step];
  v = lp_block_sum(v, red);
  if (threadIdx.x == 0) loss[0] = (float)(v / P);
}

// ---------------------------------------------------------------------------- policy loss
struct PolicyArgs {
  float low, high, kl, grad_scale;
  double log_low, log_high;  // log(1 - low), log(1 + high)
  int adv_per_token, by_sequence;
};

// e^q - q - 1, never negative. Next to 0, where the difference of e^q - 1 and q would keep nothing of q^2 / 2, from its
// series; the ninth term is 2e-9 of the sum at |q| = 1/2. e = expm1(q).
__device__ __forceinline__ float kl_term(float q, float e) {
  if (!(fabsf(q) < 0.5f)) return e - q;
  float s = 1.f / 362880.f;
  s = fmaf(s, q, 1.f / 40320.f);
  s = fmaf(s, q, 1.f / 5040.f);
  s = fmaf(s, q, 1.f / 720.f);
  s = fmaf(s, q, 1.f / 120.f);
  s = fmaf(s, q, 1.f / 24.f);
  s = fmaf(s, q, 1.f / 6.f);
  s = fmaf(s, q, 0.5f);
  return q * q * s;
}

// Terms of one token from its log-probability lp: r = e^{lp - old}; -min(r A, clip(r) A); e^q - q - 1, q = ref - lp.
// The differences are taken in fp64, their exponentials in fp32 (1e-7 of a term). Whether a ratio lies past a border is
// decided, in fp64, from the log-probability as it is returned, rounded to fp32: the gradient has lp before that, the
// statistics after it, and both must count the same tokens as clipped.
struct PolicyTerms {
  float pg, kl, cut, d;  // d = d (pg + kl_coef * kl) / d lp
};
__device__ __forceinline__ PolicyTerms policy_terms(const PolicyArgs& a, double lp, float old, bool has_ref, float ref,
                                                    float adv) {
  PolicyTerms t;
  const double lr = lp - (double)old;
  const double at = (double)(float)lp - (double)old;
  const bool cut = (adv > 0.f && at > a.log_high) || (adv < 0.f && at < a.log_low);
  const float r = expf((float)lr);
  t.pg = -(cut ? (adv > 0.f ? 1.f + a.high : 1.f - a.low) : r) * adv;
  t.d = cut ? 0.f : -r * adv;
  t.cut = cut ? 1.f : 0.f;
  t.kl = 0.f;
  if (has_ref) {
    const float q = (float)((double)ref - lp), e = expm1f(q);
    t.kl = kl_term(q, e);
    t.d -= a.kl * e;
  }
  return t;
}
// A token's weight in the loss; n: scored tokens of its sequence, total: of the batch, or its nonempty sequences.
__device__ __forceinline__ float policy_weight(const PolicyArgs& a, int n, int total) {
  return a.by_sequence ? 1.f / ((float)n * (float)total) : 1.f / (float)total;
}

// scored tokens of each sequence: a warp a sequence, or for long ones a CTA
__global__ void __launch_bounds__(256) policy_count_kernel(const long long* __restrict__ labels, long long ignore_index,
                                                           int V, int B, int T, int by_warp, int* __restrict__ counts) {
  griddep_wait();
  griddep_launch();
  __shared__ int red[8];
  const long long b = by_warp ? (long long)blockIdx.x * 8 + (threadIdx.x >> 5) : (long long)blockIdx.x;
  const int step = by_warp ? 32 : 256;
  int c = 0;
  if (b < B)
    for (int t = threadIdx.x % step; t < T; t += step) c += lp_scored(labels[b * T + t], ignore_index, V) ? 1 : 0;
  c = by_warp ? __reduce_add_sync(0xffffffffu, c) : lp_block_sum(c, red);
  if (b < B && threadIdx.x % step == 0) counts[b] = c;
}

// Sum of counts (token mean) or number of nonempty sequences (sequence mean), over the whole CTA.
__device__ __forceinline__ int policy_total(const int* __restrict__ counts, int B, int by_sequence, int* red) {
  int c = 0;
  for (int b = threadIdx.x; b < B; b += blockDim.x) c += by_sequence ? (counts[b] > 0 ? 1 : 0) : counts[b];
  return lp_block_sum(c, red);
}

__global__ void __launch_bounds__(1024) policy_total_kernel(const int* __restrict__ counts, int B, int by_sequence,
                                                            int* __restrict__ total) {
  griddep_wait();
  griddep_launch();
  __shared__ int red[32];
  const int t = policy_total(counts, B, by_sequence, red);
  if (threadIdx.x == 0) *total = t;
}

// The inputs and outputs of one row of the policy loss.
struct PolicyRows {
  const long long* labels;
  long long ignore_index;
  const float *old, *ref, *adv;
  int* counts;
  const int* total;   // policy_total, or with
  int B, count_here;  // few tokens: each CTA counts for itself, and a sequence's first CTA writes counts
  PolicyArgs a;
  float *logps, *lse, *coef;
};

// A token's inputs, loaded before its row is.
struct PolicyIn {
  float old, ref, adv;
  __device__ __forceinline__ PolicyIn(const PolicyRows& p, LpRows lr, long long row)
      : old(p.old[row]), ref(p.ref ? p.ref[row] : 0.f), adv(p.adv[p.a.adv_per_token ? row : lr.batch(row)]) {}
};
// What thread 0 does with a row's sum: the token's terms, the outputs, and the row's coefficient for the CTA.
__device__ __forceinline__ float policy_row(const PolicyRows& p, const PolicyIn& in, long long row, float xl,
                                            const LpRow& r, int n, int total, bool first) {
  const double lp = lp_label(xl, r);
  const PolicyTerms t = policy_terms(p.a, lp, in.old, p.ref != nullptr, in.ref, in.adv);
  const float coef = t.d * policy_weight(p.a, n, total) * p.a.grad_scale;
  if (first) {
    p.logps[row] = (float)lp;
    if (p.lse) p.lse[row] = (float)r.lse;
    if (p.coef) p.coef[row] = coef;
  }
  return coef;
}
// (scored tokens of the row's sequence, policy_total) over the whole CTA.
__device__ __forceinline__ int2 policy_counts(const PolicyRows& p, LpRows lr, int V, long long row, bool writer,
                                              int* red) {
  const unsigned b = lr.batch(row);
  int2 c = make_int2(0, 0);
  if (!p.count_here) return make_int2(p.counts[b], *p.total);
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (p.a.by_sequence) {  // a warp a sequence
    for (unsigned s = threadIdx.x >> 5; s < (unsigned)p.B; s += warps) {
      int n = 0;
      for (int t = lane; t < lr.T; t += 32) n += lp_scored(p.labels[(long long)s * lr.T + t], p.ignore_index, V) ? 1 : 0;
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) c.y += n > 0 ? 1 : 0, c.x += s == b ? n : 0;
    }
  } else {
    for (unsigned i = threadIdx.x; i < (unsigned)p.B * (unsigned)lr.T; i += blockDim.x) {
      const int n = lp_scored(p.labels[i], p.ignore_index, V) ? 1 : 0;
      c.y += n;
      c.x += i / (unsigned)lr.T == b ? n : 0;
    }
  }
  c.y = lp_block_sum(c.y, red);
  c.x = lp_block_sum(c.x, red);
  if (writer && threadIdx.x == 0 && (unsigned)row == b * (unsigned)lr.T) p.counts[b] = c.x;
  return c;
}
__device__ __forceinline__ void policy_row_unscored(const PolicyRows& p, long long row) {
  p.logps[row] = 0.f;
  if (p.lse) p.lse[row] = 0.f;
  if (p.coef) p.coef[row] = 0.f;
}

// A row's sum, its coefficient, then its gradient from a second read. Here for short rows, by one CTA or one warp each.
template <typename E, int W>
__global__ void __launch_bounds__(LP_THREADS) policy_kernel(const E* logits, LpRows lr, int V, const PolicyRows p,
                                                            E* dlogits, LpRows dr, long long M) {
  griddep_wait();
  griddep_launch();
  __shared__ int red[LP_THREADS / 32];
  __shared__ float s_coef;
  const LpShare sh = {0, 1};
  const long long row = lp_row<W>(sh);
  if (row >= M) return;  // whole warps
  const long long label = p.labels[row];
  const bool first = lp_rank<W>() == 0;
  E* d = dlogits ? dlogits + dr.offset(row) : nullptr;
  if (!lp_scored(label, p.ignore_index, V)) {
    if (first) policy_row_unscored(p, row);
    if (W != LP_WARP && p.count_here && (unsigned)row % (unsigned)lr.T == 0)
      policy_counts(p, lr, V, row, true, red);
    if (d) lp_write_zero<E, W>(d, V, sh);
    return;
  }
  const E* x = logits + lr.offset(row);
  const float xl = LpType<E>::get(x[label]);  // before an in-place gradient
  const PolicyIn in(p, lr, row);
  const int2 n = W == LP_WARP ? make_int2(p.counts[lr.batch(row)], *p.total) : policy_counts(p, lr, V, row, true, red);
  const LpRow r = lp_row_sum<E, W>(x, V);
  float coef = 0.f;
  if (first) coef = policy_row(p, in, row, xl, r, n.x, n.y, true);
  if (!d) return;
  if constexpr (W == LP_WARP) {
    coef = __shfl_sync(0xffffffffu, coef, 0);
  } else {
    if (threadIdx.x == 0) s_coef = coef;
    __syncthreads();
    coef = s_coef;
  }
  lp_write_grad<E, W, true>(x, d, V, (int)label, coef, sh, LpProb(r.a, r.b, -coef * r.inv));
}

// The same for long rows, by one CTA each (or a share of it), both reads by bulk copies. The second goes backwards: what
// the first read last is still in shared memory (all of a share that fits three pieces), and the rest it finds in L2 as
// long as few rows are on their way, four CTAs an SM. 16368 rows of 50304 bf16 logits, 10000 of them scored: 459 us, 5.8
// TB/s; 465 with plain loads for the second read; pieces of 8 KB, two slots or four 470 to 490. 64 such rows, a cluster
// of four CTAs each: 12.9 us, 14.0 with plain loads. Holding whole rows of this length allows two an SM, too few to cover
// their phases' latencies: 90 us more at best.
constexpr int POL_VECS = 1024, POL_SLOTS = 3;
constexpr uint32_t POL_SMEM = POL_SLOTS * POL_VECS * 16u;
template <typename E, int W>
__global__ void __launch_bounds__(LP_THREADS, 4) policy_staged_kernel(const E* logits, LpRows lr, int V,
                                                                    const PolicyRows p, E* dlogits, LpRows dr) {
  using L = LpType<E>;
  extern __shared__ __align__(128) uint8_t lp_smem[];
  __shared__ uint64_t full[POL_SLOTS];
  __shared__ int red[LP_THREADS / 32];
  __shared__ float s_coef;
  griddep_wait();
  griddep_launch();
  const LpShare sh = lp_share<W>();
  const long long row = blockIdx.x / sh.parts;
  const long long label = p.labels[row];
  E* d = dlogits ? dlogits + dr.offset(row) : nullptr;
  if (!lp_scored(label, p.ignore_index, V)) {
    if (threadIdx.x == 0 && sh.part == 0) policy_row_unscored(p, row);
    if (p.count_here && sh.part == 0 && (unsigned)row % (unsigned)lr.T == 0) policy_counts(p, lr, V, row, true, red);
    if (d) lp_write_zero<E, W>(d, V, sh);
    return;
  }
  const E* x = logits + lr.offset(row);
  const float xl = L::get(x[label]);
  const PolicyIn in(p, lr, row);
  LpRow r;
  int2 n;
  auto st = lp_stage<POL_VECS>(x, V, sh, lp_smem, full, POL_SLOTS, false);
  lp_staged_sum<E, W, LP_THREADS>(st, x, V, sh, &r, [&] {
    n = policy_counts(p, lr, V, row, sh.part == 0, red);  // while the first pieces are on their way
  });
  if (threadIdx.x == 0) s_coef = policy_row(p, in, row, xl, r, n.x, n.y, sh.part == 0);
  if (!d) return;
  __syncthreads();
  const float coef = s_coef;
  const LpProb prob(r.a, r.b, -coef * r.inv);
  if (lp_aligned(x, d)) lp_staged_grad<E, LP_THREADS>(st, x, d, V, (int)label, coef, sh, prob);
  else lp_write_grad<E, W, true>(x, d, V, (int)label, coef, sh, prob);
}

// stats = {loss, policy term, KL, clipped share}: weighted sums over the tokens, from their log-probabilities, by one CTA
// or, for many tokens, the CTAs of one cluster. total may lie in stats, which is written last.
__global__ void __launch_bounds__(1024) policy_stats_kernel(const float* __restrict__ logps,
                                                            const long long* __restrict__ labels,
                                                            long long ignore_index, int V, int B, int T,
                                                            const float* __restrict__ old, const float* __restrict__ ref,
                                                            const float* __restrict__ adv, PolicyArgs a,
                                                            const int* __restrict__ counts, const int* total_at,
                                                            float* stats) {
  griddep_wait();
  griddep_launch();
  __shared__ double3 red[32];
  __shared__ __align__(8) double mine[4];
  __shared__ int ired[32];
  const int total = total_at ? *total_at : policy_total(counts, B, a.by_sequence, ired);
  double pg = 0.0, kl = 0.0, cut = 0.0;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < (long long)B * T;
       i += (long long)gridDim.x * blockDim.x) {
    if (!lp_scored(labels[i], ignore_index, V)) continue;
    const unsigned b = (unsigned)i / (unsigned)T;
    const PolicyTerms t = policy_terms(a, (double)logps[i], old[i], ref != nullptr, ref ? ref[i] : 0.f,
                                       adv[a.adv_per_token ? i : b]);
    const double w = (double)policy_weight(a, counts[b], total);
    pg += w * (double)t.pg;
    kl += w * (double)t.kl;
    cut += w * (double)t.cut;
  }
  double3 t = lp_block_sum3(make_double3(pg, kl, cut), red);
  if (gridDim.x > 1) {
    if (threadIdx.x == 0) mine[0] = t.x, mine[1] = t.y, mine[2] = t.z;
    cluster_sync_all();
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      t = make_double3(0.0, 0.0, 0.0);
      for (unsigned c = 0; c < gridDim.x; ++c) {
        double v[3];
        for (int k = 0; k < 3; ++k) {
          const float2 h = ld_shared_cluster_f2(mapa_shared(smem_u32(&mine[k]), c));
          v[k] = __hiloint2double(__float_as_int(h.y), __float_as_int(h.x));
        }
        t.x += v[0], t.y += v[1], t.z += v[2];
      }
    }
    cluster_sync_all();  // no CTA leaves while its sums are read
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    stats[0] = (float)(t.x + (double)a.kl * t.y);
    stats[1] = (float)t.x;
    stats[2] = (float)t.y;
    stats[3] = (float)t.z;
  }
}

}  // namespace rgpt

using namespace rgpt;

// ---------------------------------------------------------------------------- host side
// Arguments that every entry point shares.
static int lp_check(const char* what, const void* logits, int dtype, long long B, long long T, int V,
                    const long long* labels) {
  int dev = 0;
  cudaGetDevice(&dev);
  const int st = rgpt_check_device(dev);
  if (st) return st;
  if (dtype < RGPT_DTYPE_BF16 || dtype > RGPT_DTYPE_F32)
    return rgpt_set_error(RGPT_ERR_BAD_SHAPE, "%s: unknown logits type %d", what, dtype);
  if (B < 1 || T < 1 || V < 1 || V > (1 << 30) || B * T > 0x7fffffffll)
    return rgpt_set_error(RGPT_ERR_BAD_SHAPE, "%s needs 1 <= B * T < 2^31 rows and 1 <= V <= 2^30 (got B=%lld T=%lld V=%d)",
                          what, B, T, V);
  if (logits == nullptr || labels == nullptr) return rgpt_set_error(RGPT_ERR_BAD_SHAPE, "%s: null pointer", what);
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == RGPT_DTYPE_F32 ? 4 : 2) != 0)
    return rgpt_set_error(RGPT_ERR_MISALIGNED, "%s: logits are not aligned to their type", what);
  return RGPT_OK;
}

template <typename F>
static void lp_dispatch(int dtype, F&& f) {
  if (dtype == RGPT_DTYPE_BF16) f((__nv_bfloat16*)nullptr);
  else if (dtype == RGPT_DTYPE_F16) f((__half*)nullptr);
  else f((float*)nullptr);
}

// CTAs a row: doubled (up to the portable cluster of 8) while the grid stays within two CTAs an SM and each part keeps
// at least 8 KB of the row. Rows of 100 KB, us for 1 / 2 / 4 / 8 CTAs a row, forward: 16 rows 8.5 / 6.8 / 5.7 / 5.2, 64 rows
// 9.6 / 7.7 / 6.9 / 6.9, 148 rows 9.9 / 8.6 / 10.3 / 12.6, 300 rows 12.4 / 12.4 / 15.3 / 19.8; policy loss: 15.0 / 13.3 / 11.8 /
// 11.5, 15.9 / 14.6 / 14.3 / 22.0, 16.8 / 18.0 / 25.1 / 37.6, 25.1 / 30.9 / 38.4 / 66.9.
static int lp_parts(long long M, int V, int dtype) {
  int dev = 0;
  cudaGetDevice(&dev);
  const long long bytes = (long long)V * (dtype == RGPT_DTYPE_F32 ? 4 : 2), full = 2ll * rgpt_num_sms(dev);
  int c = 1;
  while (c < 8 && 2 * c * M <= full && bytes / (2 * c) >= 8192) c *= 2;  // 1 for rows that a warp takes
  return c;
}

// Rows worth a trip through shared memory: below 16 KB their fixed cost (barriers, the copy's latency) shows.
static bool lp_long(int V, int dtype) { return (long long)V * (dtype == RGPT_DTYPE_F32 ? 4 : 2) >= 16384; }

// A warp a row: rows of up to 4 KB, or of up to 16 KB when there are enough of them for 8 warps an SM. bf16, forward us,
// warp / CTA a row: 700 x 2000 3.0 / 4.3, 700 x 7000 6.1 / 5.6, 2000 x 4000 5.5 / 10.1, 2000 x 7000 8.1 / 12.2.
static bool lp_warps(long long M, int V, int dtype) {
  int dev = 0;
  cudaGetDevice(&dev);
  const long long bytes = (long long)V * (dtype == RGPT_DTYPE_F32 ? 4 : 2);
  return !lp_long(V, dtype) && (bytes <= 4096 || M >= 8ll * rgpt_num_sms(dev));
}
static dim3 lp_grid(long long M, bool warps, int parts) {
  return dim3((unsigned)(warps ? (M + LP_THREADS / 32 - 1) / (LP_THREADS / 32) : M * parts));
}

// Allows `kern` its dynamic shared memory on the current device (once).
template <typename K>
static int lp_smem(K kern, uint32_t bytes, bool* set) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return rgpt_set_error(RGPT_ERR_INTERNAL, "device index %d", dev);
  if (!set[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess)
      return rgpt_check_launch("row kernel shared memory");
    set[dev] = true;
  }
  return RGPT_OK;
}

static int launch_logp_fwd(const void* logits, int dtype, LpRows lr, long long M, int V, const long long* labels,
                            long long ignore_index, float* logps, float* lse, double* wide, cudaStream_t s) {
  int rc = RGPT_OK;
  lp_dispatch(dtype, [&](auto* tag) {
    using E = std::remove_pointer_t<decltype(tag)>;
    const int c = lp_parts(M, V, dtype);
    if (lp_long(V, dtype)) {
      auto kern = c > 1 ? logp_fwd_staged_kernel<E, LP_CLUSTER> : logp_fwd_staged_kernel<E, LP_CTA>;
      static bool set[2][64] = {};
      const uint32_t smem = c > 1 ? LP_FWD_SMEM<LP_CLUSTER> : LP_FWD_SMEM<LP_CTA>;
      if ((rc = lp_smem(kern, smem, set[c > 1])) == RGPT_OK)
        launch_pdl(kern, dim3((unsigned)(M * c)), dim3(LP_FWD_THREADS), smem, s, c, (const E*)logits, lr, V, labels,
                   ignore_index, logps, lse, wide);
      return;
    }
    const bool warps = lp_warps(M, V, dtype);
    launch_pdl(warps ? logp_fwd_kernel<E, LP_WARP> : logp_fwd_kernel<E, LP_CTA>, lp_grid(M, warps, 1), dim3(LP_THREADS), 0, s,
               1, (const E*)logits, lr, V, labels, ignore_index, logps, lse, wide, M);
  });
  return rc;
}

static int launch_logp_bwd(const void* logits, int dtype, LpRows lr, long long M, int V, const long long* labels,
                            long long ignore_index, const float* lse, const float* coef, int per_seq, void* dlogits,
                            LpRows dr, cudaStream_t s) {
  lp_dispatch(dtype, [&](auto* tag) {
    using E = std::remove_pointer_t<decltype(tag)>;
    const int c = lp_parts(M, V, dtype);
    const bool warps = lp_warps(M, V, dtype);
    auto kern = warps ? logp_bwd_kernel<E, LP_WARP> : c > 1 ? logp_bwd_kernel<E, LP_CLUSTER> : logp_bwd_kernel<E, LP_CTA>;
    launch_pdl(kern, lp_grid(M, warps, c), dim3(LP_THREADS), 0, s, c, (const E*)logits, lr, V, labels, ignore_index, lse,
               coef, per_seq, (E*)dlogits, dr, M);
  });
  return RGPT_OK;
}

extern "C" int rgpt_token_logprobs(const void* logits, int dtype, long long sb, long long st, int B, int T, int V,
                                   const long long* labels, long long ignore_index, float* logps, float* lse,
                                   void* stream) {
  int rc = lp_check("token_logprobs", logits, dtype, B, T, V, labels);
  if (rc) return rc;
  if (logps == nullptr) return rgpt_set_error(RGPT_ERR_BAD_SHAPE, "token_logprobs: null output");
  rc = launch_logp_fwd(logits, dtype, LpRows{sb, st, T}, (long long)B * T, V, labels, ignore_index, logps, lse, nullptr,
                       reinterpret_cast<cudaStream_t>(stream));
  return rc ? rc : rgpt_check_launch("token_logprobs kernel");
}

extern "C" int rgpt_token_logprobs_bwd(const void* logits, int dtype, long long sb, long long st, int B, int T, int V,
                                       const long long* labels, long long ignore_index, const float* lse,
                                       const float* dlogps, void* dlogits, long long db, long long dt, void* stream) {
  int rc = lp_check("token_logprobs_bwd", logits, dtype, B, T, V, labels);
  if (rc) return rc;
  if (lse == nullptr || dlogps == nullptr || dlogits == nullptr)
    return rgpt_set_error(RGPT_ERR_BAD_SHAPE, "token_logprobs_bwd: null pointer");
  rc = launch_logp_bwd(logits, dtype, LpRows{sb, st, T}, (long long)B * T, V, labels, ignore_index, lse, dlogps, 0, dlogits,
                       LpRows{db, dt, T}, reinterpret_cast<cudaStream_t>(stream));
  return rc ? rc : rgpt_check_launch("token_logprobs_bwd kernel");
}

extern "C" int rgpt_preference_loss(const void* logits, int dtype, long long sb, long long st, int P, int T, int V,
                                    const long long* labels, long long ignore_index, const float* ref_logps, int kind,
                                    float beta, float margin, float label_smoothing, int average, float grad_scale,
                                    float* token_logps, float* lse, float* seq_logps, float* margins, float* coef,
                                    float* loss, double* scratch, void* dlogits, long long db, long long dt,
                                    void* stream) {
  int rc = lp_check("preference_loss", logits, dtype, 2ll * P, T, V, labels);
  if (rc) return rc;
  if (!token_logps || !lse || !seq_logps || !margins || !coef || !loss || !scratch)
    return rgpt_set_error(RGPT_ERR_BAD_SHAPE, "preference_loss: null output");
  if (kind < RGPT_PREF_SIGMOID || kind > RGPT_PREF_SQUARED)
    return rgpt_set_error(RGPT_ERR_BAD_SHAPE, "preference_loss: unknown kind %d", kind);
  const PrefArgs a = {kind, beta, margin, label_smoothing, grad_scale, average};
  const LpRows lr = {sb, st, T};
  const long long M = 2ll * P * T;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if ((rc = launch_logp_fwd(logits, dtype, lr, M, V, labels, ignore_index, token_logps, lse, scratch, s))) return rc;
  // A warp a pair up to 256 tokens (all three or four launches, bf16, pairs x tokens x vocabulary: 8 x 16 x 1000 7.9 us,
  // 512 x 1 x 256 10.7, 1 x 256 x 2048 10.8; one CTA going through the pairs 20.6, 833, 10.1; at 512 tokens 11.6 / 10.4).
  const int by_warp = T <= 256 ? 1 : 0;
  const unsigned pair_ctas = by_warp ? (unsigned)((P + 7) / 8) : (unsigned)P;
  launch_pdl(pref_pair_kernel, dim3(pair_ctas), dim3(256), 0, s, 1, scratch, labels, ignore_index, V, P, T,
             by_warp, ref_logps, a, seq_logps, margins, coef, loss);
  if (pair_ctas > 1) launch_pdl(pref_loss_kernel, dim3(1), dim3(256), 0, s, 1, (const double*)scratch, P, (long long)T, loss);
  if (dlogits &&
      (rc = launch_logp_bwd(logits, dtype, lr, M, V, labels, ignore_index, lse, coef, 1, dlogits, LpRows{db, dt, T}, s)))
    return rc;
  return rgpt_check_launch("preference_loss kernels");
}

extern "C" int rgpt_policy_loss(const void* logits, int dtype, long long sb, long long st, int B, int T, int V,
                                const long long* labels, long long ignore_index, const float* old_logps,
                                const float* ref_logps, const float* advantages, int adv_per_token, float clip_low,
                                float clip_high, float kl_coef, int by_sequence, float grad_scale, float* token_logps,
                                int* counts, float* stats, float* lse, float* coef, void* dlogits, long long db,
                                long long dt, void* stream) {
  int rc = lp_check("policy_loss", logits, dtype, B, T, V, labels);
  if (rc) return rc;
  if (!old_logps || !advantages || !token_logps || !counts || !stats)
    return rgpt_set_error(RGPT_ERR_BAD_SHAPE, "policy_loss: null pointer");
  const PolicyArgs a = {clip_low, clip_high, kl_coef, grad_scale, log1p(-(double)clip_low), log1p((double)clip_high),
                        adv_per_token, by_sequence};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  // Few tokens: each CTA counts them for itself while its row is on its way, which saves two launches (2 x 512 rows of
  // 100 KB 51.6 / 55.1 us with and without, 2 x 600 of 14 KB 23.6 / 21.2; for 256 sequences of one token, a warp a
  // sequence, 30.1 / 21.7).
  const long long rows = (long long)B * T;
  const int count_here = rows <= 1024 && (!by_sequence || B <= 32) ? 1 : 0;
  const bool warps = !count_here && lp_warps(rows, V, dtype);
  int* total = count_here ? nullptr : reinterpret_cast<int*>(stats);  // kept there until the statistics replace it
  if (!count_here) {
    const int by_warp = T <= 128 ? 1 : 0;
    launch_pdl(policy_count_kernel, dim3(by_warp ? (B + 7) / 8 : B), dim3(256), 0, s, 1, labels, ignore_index, V, B, T,
               by_warp, counts);
    launch_pdl(policy_total_kernel, dim3(1), dim3(1024), 0, s, 1, (const int*)counts, B, by_sequence, total);
  }
  lp_dispatch(dtype, [&](auto* tag) {
    using E = std::remove_pointer_t<decltype(tag)>;
    const LpRows lr = {sb, st, T}, dr = {db, dt, T};
    const PolicyRows p = {labels, ignore_index, old_logps,  ref_logps, advantages,  counts, total,
                          B,      count_here,   a,          token_logps, lse,       coef};
    const int c = lp_parts(rows, V, dtype);
    if (lp_long(V, dtype)) {
      auto kern = c > 1 ? policy_staged_kernel<E, LP_CLUSTER> : policy_staged_kernel<E, LP_CTA>;
      static bool set[2][64] = {};
      if ((rc = lp_smem(kern, POL_SMEM, set[c > 1])) == RGPT_OK)
        launch_pdl(kern, dim3((unsigned)(rows * c)), dim3(LP_THREADS), POL_SMEM, s, c, (const E*)logits, lr, V, p, (E*)dlogits, dr);
      return;
    }
    launch_pdl(warps ? policy_kernel<E, LP_WARP> : policy_kernel<E, LP_CTA>, lp_grid(rows, warps, 1), dim3(LP_THREADS), 0, s,
               1, (const E*)logits, lr, V, p, (E*)dlogits, dr, rows);
  });
  if (rc) return rc;
  const int ctas = rows > 8192 ? 8 : 1;
  const unsigned threads = rows < 1024 ? (unsigned)((rows + 31) / 32 * 32) : 1024u;
  launch_pdl(policy_stats_kernel, dim3(ctas), dim3(threads), 0, s, ctas, (const float*)token_logps, labels, ignore_index, V,
             B, T, old_logps, ref_logps, advantages, a, (const int*)counts, (const int*)total, stats);
  return rgpt_check_launch("policy_loss kernels");
}
