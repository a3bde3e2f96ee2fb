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
  __device__ __forceinline__ long long offset(long long row) const {
    const long long b = row / T;
    return b * sb + (row - b * T) * st;
  }
};

template <typename E>
struct LpType;
template <>
struct LpType<__nv_bfloat16> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16(v); }
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 p = unpack_bf16x2(w[k]);
      f[2 * k] = p.x, f[2 * k + 1] = p.y;
    }
  }
  static __device__ __forceinline__ float max8(const uint4& u) {  // packed compares: exact
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    const float2 m = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(m.x, m.y);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
  }
};
template <>
struct LpType<__half> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      f[2 * k] = p.x, f[2 * k + 1] = p.y;
    }
  }
  static __device__ __forceinline__ float max8(const uint4& u) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
    const float2 m = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(m.x, m.y);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const __half2 h = __floats2half2_rn(f[2 * k], f[2 * k + 1]);
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
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
    f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ float max8(const uint4& u) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

__device__ __forceinline__ bool lp_scored(long long label, long long ignore_index, int V) {
  return label != ignore_index && label >= 0 && label < V;
}

// The reference point of an exponent: -inf (nothing seen yet) is replaced by 0, so that e^{-inf - 0} = 0.
__device__ __forceinline__ float lp_ref(float m) { return m == -INFINITY ? 0.f : m; }

// A running (M, sum of 2^{c x - M}) in base 2, c = fp32(log2 e): one fused multiply-add and one exponential an
// element. M = fp32(c max) is the reference itself, so its rounding leaves no error; c's own (c ln 2 = 1 - 1.3e-8) is
// corrected to first order at the end. Elements up to LP_LOW, where c x overflows, count as nothing (M = -inf). A row
// that holds nothing else, or whose |M| is so large that c max - M may be (beyond LP_WIDE its 2^-24 |M| is no longer
// small), takes lp_row_sum's careful pass: e^{x - max} after the subtraction.
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
    const float nm = fmaxf(m, lm > LP_LOW ? lm * LP_LOG2E : -INFINITY), r = lp_ref(nm);
    s *= ex2_approx(m - r);
    m = nm;
    const float2 nr = make_float2(-r, -r), l2e = make_float2(LP_LOG2E, LP_LOG2E);
    float2 a0 = make_float2(0.f, 0.f), a1 = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < U; ++k) {
      float f[L::VEC];
      L::unpack(u[k], f);
#pragma unroll
      for (int j = 0; j < L::VEC; j += 4) {
        const float2 t0 = ffma2(make_float2(f[j], f[j + 1]), l2e, nr);
        const float2 t1 = ffma2(make_float2(f[j + 2], f[j + 3]), l2e, nr);
        a0 = fadd2(a0, make_float2(ex2_approx(t0.x), ex2_approx(t0.y)));
        a1 = fadd2(a1, make_float2(ex2_approx(t1.x), ex2_approx(t1.y)));
      }
    }
    s += (a0.x + a0.y) + (a1.x + a1.y);
  }
  __device__ __forceinline__ void add(float f) {
    const float nm = fmaxf(m, f > LP_LOW ? f * LP_LOG2E : -INFINITY), r = lp_ref(nm);
    s = s * ex2_approx(m - r) + ex2_approx(fmaf(f, LP_LOG2E, -r));
    m = nm;
  }
};

// What a row's sum comes to: probabilities e^{x - lse} = 2^{c (x - a) - b} * inv. a = 0 and b = M, or after a careful
// pass a = max and b = 0; the subtraction of a 0 is exact, so one form serves both.
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

// A row is shared by the C CTAs of a cluster (C = 1: no cluster): CTA `part` takes its share of the row's 16-byte
// vectors and of the elements that lie outside them. Several CTAs a row only when there are too few rows for the SMs.
struct LpShare {
  int part, parts;
  __device__ __forceinline__ int lo(int n) const { return (int)((long long)n * part / parts); }
  __device__ __forceinline__ int hi(int n) const { return (int)((long long)n * (part + 1) / parts); }
};
template <bool CL>
__device__ __forceinline__ LpShare lp_share() {
  LpShare s = {0, 1};
  if constexpr (CL) {
    s.part = (int)cluster_ctarank();
    s.parts = (int)cluster_nctarank();
  }
  return s;
}

// LP_UNROLL vectors in flight a thread: 4 x 16 bytes x 1280 threads on an SM cover HBM's latency at its full rate.
constexpr int LP_UNROLL = 4;

// One (m, s) for the row from each thread's, by MERGE: the same in every thread of every CTA of the row, and on return
// all of them have read it.
template <bool CL, typename MERGE>
__device__ __forceinline__ float2 lp_join(float2 a, LpShare sh, MERGE&& merge) {
  __shared__ float2 sm[LP_THREADS / 32];
  __shared__ float2 all;
  for (int o = 16; o > 0; o >>= 1)
    a = merge(a, make_float2(__shfl_xor_sync(0xffffffffu, a.x, o), __shfl_xor_sync(0xffffffffu, a.y, o)));
  __syncthreads();  // an earlier join may still be read
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = a;
  __syncthreads();
  float2 r = sm[0];
#pragma unroll
  for (int w = 1; w < LP_THREADS / 32; ++w) r = merge(r, sm[w]);
  if constexpr (CL) {
    if (threadIdx.x == 0) all = r;
    cluster_sync_all();
    r = ld_shared_cluster_f2(mapa_shared(smem_u32(&all), 0));
    for (int c = 1; c < sh.parts; ++c) r = merge(r, ld_shared_cluster_f2(mapa_shared(smem_u32(&all), (uint32_t)c)));
    cluster_sync_all();  // no CTA leaves, or writes `all` again, while another still reads it
  }
  return r;
}

// The finished row from its joined (M, s).
__device__ __forceinline__ LpRow lp_finish(float2 r) {
  // lse = ln2 (M + log2 s) + (1 - c ln2) M / c; log(s) from the mantissa in [0.75, 1.5) in fp32 (absolute error 2^-25)
  // and the exponent in fp64
  constexpr double C = (double)LP_LOG2E, LN2 = 0.69314718055994530942;
  const int e = (int)((__float_as_uint(r.y) - 0x3F400000u) & 0xFF800000u) >> 23;
  const float f = __uint_as_float(__float_as_uint(r.y) - ((uint32_t)e << 23));
  const double M = (double)r.x;
  return LpRow{0.f, r.x, 1.f / r.y, fma(M, LN2 + (1.0 - C * LN2) / C, fma((double)e, LN2, (double)logf(f)))};
}
__device__ __forceinline__ bool lp_plain(float2 r) {
  return fabsf(r.x) <= LP_WIDE && r.y < INFINITY;  // a NaN in the row makes the sum NaN
}

// The careful pass over a row in global memory by n threads (index t), joined by `join` (the same in all of them).
template <typename E, typename J>
__device__ __noinline__ LpRow lp_careful(const E* x, int V, int t, int n, J join) {
  float top = -INFINITY, sum = 0.f;
  for (int j = t; j < V; j += n) top = fmaxf(top, LpType<E>::get(x[j]));
  const float ref = lp_ref(join(make_float2(top, 0.f), true).x);
  for (int j = t; j < V; j += n) sum += ex2_approx((LpType<E>::get(x[j]) - ref) * LP_LOG2E);
  sum = join(make_float2(sum, 0.f), false).x;
  return LpRow{ref, 0.f, 1.f / sum, (double)ref + log((double)sum)};
}
__device__ __forceinline__ float2 lp_merge(float2 p, float2 q) {
  LpSum t;
  t.m = p.x, t.s = p.y;
  t.merge(q.x, q.y);
  return make_float2(t.m, t.s);
}
template <bool CL>
struct LpCtaJoin {
  LpShare sh;
  __device__ float2 operator()(float2 v, bool max) const {
    return max ? lp_join<CL>(v, sh, [](float2 p, float2 q) { return make_float2(fmaxf(p.x, q.x), 0.f); })
               : lp_join<CL>(v, sh, [](float2 p, float2 q) { return make_float2(p.x + q.x, 0.f); });
  }
};

// The sum of one row, the same in every thread of its CTAs, all of which have read it on return.
template <typename E, bool CL>
__device__ __forceinline__ LpRow lp_row_sum(const E* x, int V, LpShare sh) {
  using L = LpType<E>;
  const int head = lp_head(x, V), nvec = (V - head) / L::VEC;
  LpSum a;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  int v = sh.lo(nvec) + threadIdx.x;
  const int vend = sh.hi(nvec);
  for (; v + (LP_UNROLL - 1) * LP_THREADS < vend; v += LP_UNROLL * LP_THREADS) {
    uint4 u[LP_UNROLL];
#pragma unroll
    for (int k = 0; k < LP_UNROLL; ++k) u[k] = xv[v + k * LP_THREADS];
    a.template add<L, LP_UNROLL>(u);
  }
  for (; v < vend; v += LP_THREADS) {
    const uint4 u[1] = {xv[v]};
    a.template add<L, 1>(u);
  }
  const int rest = V - nvec * L::VEC;  // the head, then the tail behind the vectors
  for (int j = sh.lo(rest) + threadIdx.x; j < sh.hi(rest); j += LP_THREADS)
    a.add(L::get(x[j < head ? j : j + nvec * L::VEC]));
  const float2 r = lp_join<CL>(make_float2(a.m, a.s), sh, lp_merge);
  if (lp_plain(r)) return lp_finish(r);
  return lp_careful(x, V, sh.part * LP_THREADS + (int)threadIdx.x, sh.parts * LP_THREADS, LpCtaJoin<CL>{sh});
}

// This CTA's share of coef * ([j = label] - p(x_j)) over one row; prob maps two logits to two probabilities. d may be
// x: each thread reads an element before it writes the same one.
template <typename E, typename P>
__device__ __forceinline__ void lp_write_grad(const E* x, E* d, int V, int label, float coef, LpShare sh, P&& prob) {
  using L = LpType<E>;
  const bool vec = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
  const int head = vec ? lp_head(x, V) : V, nvec = (V - head) / L::VEC;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  uint4* dv = reinterpret_cast<uint4*>(d + head);
  const float2 nc = make_float2(-coef, -coef);
  auto one = [&](const uint4& u, int at) {
    float f[L::VEC];
    L::unpack(u, f);
#pragma unroll
    for (int k = 0; k < L::VEC; k += 2) {
      const float2 g = fmul2(prob(make_float2(f[k], f[k + 1])), nc);
      f[k] = g.x, f[k + 1] = g.y;
    }
    if (at >= 0 && at < L::VEC) {
#pragma unroll
      for (int k = 0; k < L::VEC; ++k) f[k] += k == at ? coef : 0.f;
    }
    return L::pack(f);
  };
  int v = sh.lo(nvec) + threadIdx.x;
  const int vend = sh.hi(nvec);
  for (; v + (LP_UNROLL - 1) * LP_THREADS < vend; v += LP_UNROLL * LP_THREADS) {
    uint4 u[LP_UNROLL];
#pragma unroll
    for (int k = 0; k < LP_UNROLL; ++k) u[k] = xv[v + k * LP_THREADS];
#pragma unroll
    for (int k = 0; k < LP_UNROLL; ++k)
      dv[v + k * LP_THREADS] = one(u[k], label - head - (v + k * LP_THREADS) * L::VEC);
  }
  for (; v < vend; v += LP_THREADS) dv[v] = one(xv[v], label - head - v * L::VEC);
  const int rest = V - nvec * L::VEC;
  for (int i = sh.lo(rest) + threadIdx.x; i < sh.hi(rest); i += LP_THREADS) {
    const int j = i < head ? i : i + nvec * L::VEC;
    const float p = prob(make_float2(L::get(x[j]), 0.f)).x;
    d[j] = L::put(j == label ? coef - coef * p : -coef * p);
  }
}

template <typename E>
__device__ __forceinline__ void lp_write_zero(E* d, int V, LpShare sh) {
  using L = LpType<E>;
  const int head = lp_head(d, V), nvec = (V - head) / L::VEC;
  uint4* dv = reinterpret_cast<uint4*>(d + head);
  for (int v = sh.lo(nvec) + threadIdx.x; v < sh.hi(nvec); v += LP_THREADS) dv[v] = make_uint4(0u, 0u, 0u, 0u);
  const int rest = V - nvec * L::VEC;
  for (int i = sh.lo(rest) + threadIdx.x; i < sh.hi(rest); i += LP_THREADS)
    d[i < head ? i : i + nvec * L::VEC] = L::put(0.f);
}

// 2^{c (x - a) - b} of two logits, times a factor
struct LpProb {
  float2 na, nb, k;
  __device__ __forceinline__ LpProb(float a, float b, float factor)
      : na(make_float2(-a, -a)), nb(make_float2(-b, -b)), k(make_float2(factor, factor)) {}
  __device__ __forceinline__ float2 operator()(float2 f) const {
    const float2 t = ffma2(fadd2(f, na), make_float2(LP_LOG2E, LP_LOG2E), nb);
    return fmul2(make_float2(ex2_approx(t.x), ex2_approx(t.y)), k);
  }
};

// ---------------------------------------------------------------------------- token log-probabilities
// One pass over a row with a running maximum and sum.
template <typename E, bool CL>
__global__ void __launch_bounds__(LP_THREADS) logp_fwd_kernel(const E* __restrict__ logits, LpRows lr, int V,
                                                              const long long* __restrict__ labels,
                                                              long long ignore_index, float* __restrict__ logps,
                                                              float* __restrict__ lse, double* __restrict__ wide) {
  griddep_wait();
  griddep_launch();
  const LpShare sh = lp_share<CL>();
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
  const LpRow r = lp_row_sum<E, CL>(x, V, sh);
  if (first) {
    const double lp = (double)LpType<E>::get(x[label]) - r.lse;
    logps[row] = (float)lp;
    if (lse) lse[row] = (float)r.lse;
    if (wide) wide[row] = lp;
  }
}

// dlogits = coef * (onehot - e^{x - lse}); coef per token, or per sequence (per_seq). Elementwise, so dlogits may be
// the logits themselves.
template <typename E, bool CL>
__global__ void __launch_bounds__(LP_THREADS) logp_bwd_kernel(const E* logits, LpRows lr, int V,
                                                              const long long* __restrict__ labels,
                                                              long long ignore_index, const float* __restrict__ lse,
                                                              const float* __restrict__ coef, int per_seq, E* dlogits,
                                                              LpRows dr) {
  griddep_wait();
  griddep_launch();
  const LpShare sh = lp_share<CL>();
  const long long row = blockIdx.x / sh.parts;
  const long long label = labels[row];
  E* d = dlogits + dr.offset(row);
  if (!lp_scored(label, ignore_index, V)) {
    lp_write_zero(d, V, sh);
    return;
  }
  const E* x = logits + lr.offset(row);
  const float l = lse[row], c = coef[per_seq ? row / lr.T : row];
  LpRow r = {l, 0.f, 1.f, 0.0};
  if (!(fabsf(l) <= LP_LSE_EXACT)) {
    r = lp_careful(x, V, sh.part * LP_THREADS + (int)threadIdx.x, sh.parts * LP_THREADS, LpCtaJoin<CL>{sh});
    __syncthreads();  // every thread has read the row before an in-place gradient
  }
  lp_write_grad(x, d, V, (int)label, c, sh, LpProb(r.a, r.b, r.inv));
}

// ---------------------------------------------------------------------------- sums over a CTA
__device__ __forceinline__ double lp_block_sum(double v, double* red) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();  // red may still be read from an earlier sum
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) t += red[w];
  return t;
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

// One CTA per pair: the two sequences' log-probabilities in fp64, the margin h and the sequences' coefficients
// d loss / d (a scored token's log-probability).
__global__ void __launch_bounds__(256) pref_pair_kernel(const double* __restrict__ logps,
                                                        const long long* __restrict__ labels, long long ignore_index,
                                                        int V, int P, int T, const float* __restrict__ ref, PrefArgs a,
                                                        float* __restrict__ seq_logps, float* __restrict__ margins,
                                                        float* __restrict__ coef) {
  griddep_wait();
  griddep_launch();
  __shared__ double red[8];
  const int p = blockIdx.x;
  double s[2], n[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const long long base = (long long)(p + k * P) * T;
    double v = 0.0, c = 0.0;
    for (int t = threadIdx.x; t < T; t += blockDim.x) {
      v += logps[base + t];
      if (a.average) c += lp_scored(labels[base + t], ignore_index, V) ? 1.0 : 0.0;
    }
    s[k] = lp_block_sum(v, red);
    n[k] = a.average ? fmax(lp_block_sum(c, red), 1.0) : 1.0;
    s[k] /= n[k];
  }
  if (threadIdx.x != 0) return;
  double d = s[0] - s[1];
  if (ref) d = (s[0] - (double)ref[p]) - (s[1] - (double)ref[p + P]);
  const double h = (double)a.beta * d - (double)a.margin;
  double loss, dh;
  pref_terms(a, h, &loss, &dh);
  dh *= (double)a.beta * (double)a.grad_scale / P;
  seq_logps[p] = (float)s[0];
  seq_logps[p + P] = (float)s[1];
  margins[p] = (float)h;
  coef[p] = (float)(dh / n[0]);
  coef[p + P] = (float)(-dh / n[1]);
}

// mean of the pairs' losses, from their margins
__global__ void __launch_bounds__(256) pref_loss_kernel(const float* __restrict__ margins, int P, PrefArgs a,
                                                        float* __restrict__ loss) {
  griddep_wait();
  griddep_launch();
  __shared__ double red[8];
  double v = 0.0;
  for (int p = threadIdx.x; p < P; p += blockDim.x) {
    double l, dh;
    pref_terms(a, (double)margins[p], &l, &dh);
    v += l;
  }
  v = lp_block_sum(v, red);
  if (threadIdx.x == 0) loss[0] = (float)(v / P);
}

// ---------------------------------------------------------------------------- policy loss
struct PolicyArgs {
  float low, high, kl, grad_scale;
  int adv_per_token, by_sequence;
};

// Terms of one token from its log-probability lp: r = e^{lp - old}; -min(r A, clip(r) A); e^q - q - 1, q = ref - lp.
struct PolicyTerms {
  double pg, kl, cut, d;  // d = d (pg + kl_coef * kl) / d lp
};
__device__ __forceinline__ PolicyTerms policy_terms(const PolicyArgs& a, double lp, double old, bool has_ref, double ref,
                                                    double adv) {
  PolicyTerms t;
  const double r = exp(lp - old);
  const double hi = 1.0 + (double)a.high, lo = 1.0 - (double)a.low;
  const bool cut = (adv > 0.0 && r > hi) || (adv < 0.0 && r < lo);
  t.pg = cut ? -(adv > 0.0 ? hi : lo) * adv : -r * adv;
  t.d = cut ? 0.0 : -r * adv;
  t.cut = cut ? 1.0 : 0.0;
  t.kl = 0.0;
  if (has_ref) {
    const double q = ref - lp, e = exp(q);
    t.kl = e - q - 1.0;
    t.d += (double)a.kl * (1.0 - e);
  }
  return t;
}

// scored tokens of each sequence
__global__ void __launch_bounds__(256) policy_count_kernel(const long long* __restrict__ labels, long long ignore_index,
                                                           int V, int T, int* __restrict__ counts) {
  griddep_wait();
  griddep_launch();
  __shared__ double red[8];
  const long long base = (long long)blockIdx.x * T;
  double c = 0.0;
  for (int t = threadIdx.x; t < T; t += blockDim.x) c += lp_scored(labels[base + t], ignore_index, V) ? 1.0 : 0.0;
  c = lp_block_sum(c, red);
  if (threadIdx.x == 0) counts[blockIdx.x] = (int)c;
}

// Sum of counts (token mean) or number of nonempty sequences (sequence mean), over the whole CTA.
__device__ __forceinline__ double policy_total(const int* __restrict__ counts, int B, int by_sequence, double* red) {
  double c = 0.0;
  for (int b = threadIdx.x; b < B; b += blockDim.x) c += by_sequence ? (counts[b] > 0 ? 1.0 : 0.0) : (double)counts[b];
  return lp_block_sum(c, red);
}

template <typename E, bool CL>
__global__ void __launch_bounds__(LP_THREADS) policy_kernel(const E* logits, LpRows lr, int B, int V,
                                                            const long long* __restrict__ labels,
                                                            long long ignore_index, const float* __restrict__ old,
                                                            const float* __restrict__ ref, const float* __restrict__ adv,
                                                            PolicyArgs a, const int* __restrict__ counts,
                                                            float* __restrict__ logps, float* __restrict__ lse,
                                                            float* __restrict__ coef, E* dlogits, LpRows dr) {
  griddep_wait();
  griddep_launch();
  __shared__ double red[LP_THREADS / 32];
  __shared__ float s_coef;
  const LpShare sh = lp_share<CL>();
  const long long row = blockIdx.x / sh.parts;
  const long long label = labels[row];
  const bool first = threadIdx.x == 0 && sh.part == 0;
  E* d = dlogits ? dlogits + dr.offset(row) : nullptr;
  if (!lp_scored(label, ignore_index, V)) {
    if (first) {
      logps[row] = 0.f;
      if (lse) lse[row] = 0.f;
      if (coef) coef[row] = 0.f;
    }
    if (d) lp_write_zero(d, V, sh);
    return;
  }
  const E* x = logits + lr.offset(row);
  const float xl = LpType<E>::get(x[label]);  // before an in-place gradient
  const double total = policy_total(counts, B, a.by_sequence, red);
  const LpRow r = lp_row_sum<E, CL>(x, V, sh);
  if (threadIdx.x == 0) {
    const double lp = (double)xl - r.lse;
    const long long b = row / lr.T;
    const PolicyTerms t = policy_terms(a, lp, (double)old[row], ref != nullptr, ref ? (double)ref[row] : 0.0,
                                       (double)adv[a.adv_per_token ? row : b]);
    const double w = a.by_sequence ? 1.0 / ((double)counts[b] * total) : 1.0 / total;
    s_coef = (float)(t.d * w * (double)a.grad_scale);
    if (first) {
      logps[row] = (float)lp;
      if (lse) lse[row] = (float)r.lse;
      if (coef) coef[row] = s_coef;
    }
  }
  if (!d) return;
  __syncthreads();
  lp_write_grad(x, d, V, (int)label, s_coef, sh, LpProb(r.a, r.b, r.inv));
}

// stats = {loss, policy term, KL, clipped share}: weighted sums over the tokens, from their log-probabilities
__global__ void __launch_bounds__(1024) policy_stats_kernel(const float* __restrict__ logps,
                                                            const long long* __restrict__ labels,
                                                            long long ignore_index, int V, int B, int T,
                                                            const float* __restrict__ old, const float* __restrict__ ref,
                                                            const float* __restrict__ adv, PolicyArgs a,
                                                            const int* __restrict__ counts, float* __restrict__ stats) {
  griddep_wait();
  griddep_launch();
  __shared__ double red[32];
  const double total = policy_total(counts, B, a.by_sequence, red);
  double pg = 0.0, kl = 0.0, cut = 0.0;
  for (long long i = threadIdx.x; i < (long long)B * T; i += blockDim.x) {
    if (!lp_scored(labels[i], ignore_index, V)) continue;
    const long long b = i / T;
    const PolicyTerms t = policy_terms(a, (double)logps[i], (double)old[i], ref != nullptr, ref ? (double)ref[i] : 0.0,
                                       (double)adv[a.adv_per_token ? i : b]);
    const double w = a.by_sequence ? 1.0 / ((double)counts[b] * total) : 1.0 / total;
    pg += w * t.pg;
    kl += w * t.kl;
    cut += w * t.cut;
  }
  pg = lp_block_sum(pg, red);
  kl = lp_block_sum(kl, red);
  cut = lp_block_sum(cut, red);
  if (threadIdx.x == 0) {
    stats[0] = (float)(pg + (double)a.kl * kl);
    stats[1] = (float)pg;
    stats[2] = (float)kl;
    stats[3] = (float)cut;
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
  if (B < 1 || T < 1 || V < 1 || B * T > 0x7fffffffll)
    return rgpt_set_error(RGPT_ERR_BAD_SHAPE, "%s needs 1 <= B * T < 2^31 rows and V >= 1 (got B=%lld T=%lld V=%d)", what,
                          B, T, V);
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

// CTAs a row: doubled (up to the portable cluster of 8) while the grid leaves SMs without their share of CTAs and each
// part keeps at least 8 KB of the row.
static int lp_parts(long long M, int V, int dtype) {
  int dev = 0;
  cudaGetDevice(&dev);
  const long long bytes = (long long)V * (dtype == RGPT_DTYPE_F32 ? 4 : 2), full = 4ll * rgpt_num_sms(dev);
  int c = 1;
  while (c < 8 && 2 * c * M <= full && bytes / (2 * c) >= 8192) c *= 2;
  return c;
}

static void launch_logp_fwd(const void* logits, int dtype, LpRows lr, long long M, int V, const long long* labels,
                            long long ignore_index, float* logps, float* lse, double* wide, cudaStream_t s) {
  lp_dispatch(dtype, [&](auto* tag) {
    using E = std::remove_pointer_t<decltype(tag)>;
    const int c = lp_parts(M, V, dtype);
    launch_pdl(c > 1 ? logp_fwd_kernel<E, true> : logp_fwd_kernel<E, false>, dim3((unsigned)(M * c)), dim3(LP_THREADS), 0,
               s, c, (const E*)logits, lr, V, labels, ignore_index, logps, lse, wide);
  });
}

static void launch_logp_bwd(const void* logits, int dtype, LpRows lr, long long M, int V, const long long* labels,
                            long long ignore_index, const float* lse, const float* coef, int per_seq, void* dlogits,
                            LpRows dr, cudaStream_t s) {
  lp_dispatch(dtype, [&](auto* tag) {
    using E = std::remove_pointer_t<decltype(tag)>;
    const int c = lp_parts(M, V, dtype);
    launch_pdl(c > 1 ? logp_bwd_kernel<E, true> : logp_bwd_kernel<E, false>, dim3((unsigned)(M * c)), dim3(LP_THREADS), 0,
               s, c, (const E*)logits, lr, V, labels, ignore_index, lse, coef, per_seq, (E*)dlogits, dr);
  });
}

extern "C" int rgpt_token_logprobs(const void* logits, int dtype, long long sb, long long st, int B, int T, int V,
                                   const long long* labels, long long ignore_index, float* logps, float* lse,
                                   void* stream) {
  const int rc = lp_check("token_logprobs", logits, dtype, B, T, V, labels);
  if (rc) return rc;
  if (logps == nullptr) return rgpt_set_error(RGPT_ERR_BAD_SHAPE, "token_logprobs: null output");
  launch_logp_fwd(logits, dtype, LpRows{sb, st, T}, (long long)B * T, V, labels, ignore_index, logps, lse,
                  nullptr, reinterpret_cast<cudaStream_t>(stream));
  return rgpt_check_launch("logp_fwd_kernel");
}

extern "C" int rgpt_token_logprobs_bwd(const void* logits, int dtype, long long sb, long long st, int B, int T, int V,
                                       const long long* labels, long long ignore_index, const float* lse,
                                       const float* dlogps, void* dlogits, long long db, long long dt, void* stream) {
  const int rc = lp_check("token_logprobs_bwd", logits, dtype, B, T, V, labels);
  if (rc) return rc;
  if (lse == nullptr || dlogps == nullptr || dlogits == nullptr)
    return rgpt_set_error(RGPT_ERR_BAD_SHAPE, "token_logprobs_bwd: null pointer");
  launch_logp_bwd(logits, dtype, LpRows{sb, st, T}, (long long)B * T, V, labels, ignore_index, lse, dlogps, 0, dlogits,
                  LpRows{db, dt, T}, reinterpret_cast<cudaStream_t>(stream));
  return rgpt_check_launch("logp_bwd_kernel");
}

extern "C" int rgpt_preference_loss(const void* logits, int dtype, long long sb, long long st, int P, int T, int V,
                                    const long long* labels, long long ignore_index, const float* ref_logps, int kind,
                                    float beta, float margin, float label_smoothing, int average, float grad_scale,
                                    float* token_logps, float* lse, float* seq_logps, float* margins, float* coef,
                                    float* loss, double* scratch, void* dlogits, long long db, long long dt,
                                    void* stream) {
  const int rc = lp_check("preference_loss", logits, dtype, 2ll * P, T, V, labels);
  if (rc) return rc;
  if (!token_logps || !lse || !seq_logps || !margins || !coef || !loss || !scratch)
    return rgpt_set_error(RGPT_ERR_BAD_SHAPE, "preference_loss: null output");
  if (kind < RGPT_PREF_SIGMOID || kind > RGPT_PREF_SQUARED)
    return rgpt_set_error(RGPT_ERR_BAD_SHAPE, "preference_loss: unknown kind %d", kind);
  const PrefArgs a = {kind, beta, margin, label_smoothing, grad_scale, average};
  const LpRows lr = {sb, st, T};
  const long long M = 2ll * P * T;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  launch_logp_fwd(logits, dtype, lr, M, V, labels, ignore_index, token_logps, lse, scratch, s);
  launch_pdl(pref_pair_kernel, dim3(P), dim3(256), 0, s, 1, (const double*)scratch, labels, ignore_index, V, P, T, ref_logps, a,
             seq_logps, margins, coef);
  launch_pdl(pref_loss_kernel, dim3(1), dim3(256), 0, s, 1, margins, P, a, loss);
  if (dlogits)
    launch_logp_bwd(logits, dtype, lr, M, V, labels, ignore_index, lse, coef, 1, dlogits, LpRows{db, dt, T}, s);
  return rgpt_check_launch("preference_loss kernels");
}

extern "C" int rgpt_policy_loss(const void* logits, int dtype, long long sb, long long st, int B, int T, int V,
                                const long long* labels, long long ignore_index, const float* old_logps,
                                const float* ref_logps, const float* advantages, int adv_per_token, float clip_low,
                                float clip_high, float kl_coef, int by_sequence, float grad_scale, float* token_logps,
                                int* counts, float* stats, float* lse, float* coef, void* dlogits, long long db,
                                long long dt, void* stream) {
  const int rc = lp_check("policy_loss", logits, dtype, B, T, V, labels);
  if (rc) return rc;
  if (!old_logps || !advantages || !token_logps || !counts || !stats)
    return rgpt_set_error(RGPT_ERR_BAD_SHAPE, "policy_loss: null pointer");
  const PolicyArgs a = {clip_low, clip_high, kl_coef, grad_scale, adv_per_token, by_sequence};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  launch_pdl(policy_count_kernel, dim3(B), dim3(256), 0, s, 1, labels, ignore_index, V, T, counts);
  lp_dispatch(dtype, [&](auto* tag) {
    using E = std::remove_pointer_t<decltype(tag)>;
    const int c = lp_parts((long long)B * T, V, dtype);
    launch_pdl(c > 1 ? policy_kernel<E, true> : policy_kernel<E, false>, dim3((unsigned)((long long)B * T * c)),
               dim3(LP_THREADS), 0, s, c, (const E*)logits, LpRows{sb, st, T}, B, V, labels, ignore_index, old_logps,
               ref_logps, advantages, a, (const int*)counts, token_logps, lse, coef, (E*)dlogits, LpRows{db, dt, T});
  });
  launch_pdl(policy_stats_kernel, dim3(1), dim3(1024), 0, s, 1, (const float*)token_logps, labels, ignore_index, V, B, T,
             old_logps, ref_logps, advantages, a, (const int*)counts, stats);
  return rgpt_check_launch("policy_loss kernels");
}
