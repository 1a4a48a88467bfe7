// moe_scored.cu — expert routing by scores: softmax or sigmoid, a bias that steers the choice
// only, experts in groups of which the best are open, top-k, weights.
//
//   s = sigmoid(l)  or  softmax(l)          c = s + bias
//   group score     = best c of the group, or the sum of its two best
//   open groups     = the top_groups best;  ids = the top-k c of the open groups, in order
//   w = s[ids] (/ sum s[ids] when renorm) * scale
// Equal values go to the lower group / expert index. A NaN logit counts as -inf.
//
// One warp per token, lane i holds the EPL consecutive experts from i * EPL on, so the lowest lane
// among equals is the lowest index and a pick is one warp-wide integer max of order-preserving
// keys plus a ballot. Without a bias the choice follows the logits themselves (both scores are
// monotone in them): no rounding can reorder it. With a bias, fp32 values cut the row to a short
// list (with a margin for their error) whose exact values, one fp64 score per lane, are compared.
// Group scores are compared in fp32; where an open and a closed group lie within their own error
// bounds the same warp ranks the groups again in fp64. So the ids are those of the exact scores.
//
// What bounds a large step is instructions and their latency (16384 tokens, 256 experts in 8 groups, top
// 8, bf16: 23 us for 9.4 MB; 1114 warp instructions per token, which issue in 69 % of the cycles, the rest
// are fixed latencies and shuffles that wait for one another): scores and group sums 10 us of it, the short
// list 1, exact scores 1.4, picks 2.3, weights 3, and 4 that the few rows ranked again keep the last wave.
// Picking all 8 from 32 * EPL values, and every close row again in fp64, took 41 us.
#include "kernels.h"
#include "launch.cuh"
#include "step_ops.h"

namespace sq {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kWarps = 8;
constexpr float kNegInf = -INFINITY;

__device__ __forceinline__ uint32_t ord32(float f) {
  const uint32_t u = __float_as_uint(f);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unord32(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
// NaN -> -inf, -0 -> +0 (so that equal values have equal keys)
__device__ __forceinline__ float clean(float v) { return v == v ? v + 0.0f : kNegInf; }

__device__ __forceinline__ double score64(float x, bool sigmoid, float m, double inv_z) {
  if (sigmoid) return 1.0 / (1.0 + exp(-(double)x));
  return (x == m ? 1.0 : exp((double)x - (double)m)) * inv_z;
}

// Scores for the fp32 choice: the hardware's exponential and reciprocal (2 and 1 ulp).
__device__ __forceinline__ float exp_fast(float x) {  // x <= 0 or the score saturates: flushing is harmless
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(1.4426950408889634f * x));
  return e;
}
__device__ __forceinline__ float sigmoid_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + exp_fast(-x)));
  return r;
}

__device__ __forceinline__ float max2(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float min2(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double max2(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ double min2(double a, double b) { return fmin(a, b); }
// The two largest of (a1 >= a2) and (b1 >= b2).
template <class S>
__device__ __forceinline__ void merge2(S& a1, S& a2, S b1, S b2) {
  a2 = max2(min2(a1, b1), max2(a2, b2));
  a1 = max2(a1, b1);
}

struct Shape {
  int E, K, groups, top_groups, gsize, lanes;  // lanes: lanes per group when EPL divides the group, else 0
  bool top2;
};

// Two best values of group `lane` (lane < groups), from per-lane values v[EPL] (consecutive experts).
template <int EPL, class S>
__device__ __forceinline__ void group_top2(const S (&v)[EPL], const Shape& sh, int lane, S* buf, S& g1, S& g2) {
  const S ninf = (S)kNegInf;
  g1 = g2 = ninf;
  if (sh.lanes > 0) {
    S t1 = ninf, t2 = ninf;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      t2 = max2(t2, min2(t1, v[i]));
      t1 = max2(t1, v[i]);
    }
    S r1 = t1, r2 = t2;
    const int base = lane / sh.lanes * sh.lanes;
    for (int o = 1; o < sh.lanes; ++o) {
      int from = lane + o;
      if (from >= base + sh.lanes) from -= sh.lanes;
      const S b1 = __shfl_sync(kFull, t1, from & 31), b2 = __shfl_sync(kFull, t2, from & 31);
      merge2(r1, r2, b1, b2);
    }
    const int src = lane < sh.groups ? lane * sh.lanes : 0;
    g1 = __shfl_sync(kFull, r1, src);
    g2 = __shfl_sync(kFull, r2, src);
  } else {  // a group starts inside a lane: through shared memory, one lane per group
    __syncwarp();
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (lane * EPL + i < sh.E) buf[lane * EPL + i] = v[i];
    __syncwarp();
    if (lane < sh.groups)
      for (int i = 0; i < sh.gsize; ++i) merge2(g1, g2, buf[lane * sh.gsize + i], ninf);
  }
}

// Open groups by score (lane g < groups: gscore, off by at most err). sure: false when an open and a closed
// group's exact scores may be the other way round; err < 0: the scores are exact.
__device__ __forceinline__ unsigned open_groups32(float gscore, const Shape& sh, int lane, float err, bool& sure) {
  uint32_t gk = lane < sh.groups ? ord32(clean(gscore)) : 0u;
  unsigned open = 0;
  for (int g = 0; g < sh.top_groups; ++g) {
    const uint32_t best = __reduce_max_sync(kFull, gk);
    const int win = __ffs(__ballot_sync(kFull, gk == best)) - 1;
    open |= 1u << win;
    if (lane == win) gk = 0u;
  }
  sure = true;
  if (err >= 0.f && sh.top_groups < sh.groups) {  // (one case for the whole warp)
    // the least that an open group's score can be against the most that a closed one's can be (NaN, of an
    // infinite error: anything)
    const bool in = (open >> lane) & 1u;
    const float low = gscore - err, high = gscore + err;
    const uint32_t lo = __reduce_min_sync(kFull, in ? ord32(clean(low)) : 0xffffffffu);
    const uint32_t hi = __reduce_max_sync(kFull, !in && lane < sh.groups ? ord32(high == high ? high : INFINITY) : 0u);
    sure = lo > hi;
  }
  return open;
}

// Picks up to which the short list is used; beyond, it seldom fits the lanes (4096 tokens, 256 experts:
// 16 picks 6.9 us by the list, 17 picks 10.6 us from all values; with a bias 13.9 and 23.7 us).
constexpr int kListK = 16;

// Short list of a row: the K-th largest of the lanes' maxima is a bound that at least K values reach
// and a few more (for K = 8 about 4, for K = 16 about 5); those down to `margin` below it are laid out in index order, one per
// lane, where a pick is a maximum and a ballot. (Picking from 32 * EPL values costs every lane a new
// maximum of its EPL values per pick.) Returns their number, or 33 when they are more than the lanes.
template <int EPL>
__device__ __forceinline__ int short_list(const uint32_t (&k)[EPL], int K, float margin, int lane, uint2* cand,
                                          uint2& my) {
  uint32_t lm = 0u, bound = 0u;
#pragma unroll
  for (int i = 0; i < EPL; ++i) lm = max(lm, k[i]);
  for (int kk = 0; kk < K; ++kk) {
    bound = __reduce_max_sync(kFull, lm);
    const int win = __ffs(__ballot_sync(kFull, lm == bound)) - 1;
    if (lane == win) lm = 0u;
  }
  if (bound != 0u && margin > 0.f) {
    const float v = unord32(bound);
    if (v < INFINITY) bound = v > kNegInf ? ord32(v - margin * (1.f + fabsf(v))) : 1u;
  }
  bound = max(bound, 1u);  // (fewer open lanes than picks: every open value)
  int n = 0;
#pragma unroll
  for (int i = 0; i < EPL; ++i) n += k[i] >= bound;
  int at = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(kFull, at, o);
    if (lane >= o) at += v;
  }
  const int total = __shfl_sync(kFull, at, 31);
  if (total > 32) return 33;
  at -= n;
  if (n > 0) {
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (k[i] >= bound) cand[at++] = make_uint2(k[i], lane * EPL + i);
  }
  __syncwarp();
  my = lane < total ? cand[lane] : make_uint2(0u, 0u);
  return total;
}

// fp64 value as an order-preserving pair of words.
__device__ __forceinline__ void ord64(double v, uint32_t& hi, uint32_t& lo) {
  unsigned long long u = __double_as_longlong(v + 0.0);
  u ^= (unsigned long long)((long long)u >> 63) | 0x8000000000000000ull;
  hi = (uint32_t)(u >> 32);
  lo = (uint32_t)u;
}

// The K largest of the lanes' keys (hi, lo; hi = 0: none), in order, the lower lane first among equals:
// lane kk returns the lane of pick kk, `taken` all of them.
template <bool kTwo>
__device__ __forceinline__ int pick_list(uint32_t hi, uint32_t lo, int K, int lane, unsigned& taken) {
  int src = 0;
  taken = 0;
  for (int kk = 0; kk < K; ++kk) {
    const uint32_t m = __reduce_max_sync(kFull, hi);
    unsigned w = __ballot_sync(kFull, hi == m);
    if (kTwo && (w & (w - 1u))) {  // the upper words tie: the lower ones decide
      const uint32_t l = __reduce_max_sync(kFull, hi == m ? lo : 0u);
      w &= __ballot_sync(kFull, lo == l);
    }
    w &= 0u - w;
    taken |= w;
    if (lane == kk) src = __ffs(w) - 1;
    if ((w >> lane) & 1u) hi = 0u;
  }
  return src;
}

// The K largest of all keys, one after another (more picks, or more equal values, than a short list).
template <int EPL>
__device__ __forceinline__ int pick_all(uint32_t (&k)[EPL], int K, int lane) {
  int my_id = 0, bi = 0;
  uint32_t best = 0u;
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (k[i] > best) {
      best = k[i];
      bi = i;
    }
  for (int kk = 0; kk < K; ++kk) {
    const uint32_t m = __reduce_max_sync(kFull, best);
    const int win = __ffs(__ballot_sync(kFull, best == m)) - 1;
    const int id = win * EPL + __shfl_sync(kFull, bi, win);
    if (lane == kk) my_id = id;
    if (lane == win) {
      best = 0u;
      const int gone = bi;
      bi = 0;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        if (i == gone) k[i] = 0u;
        if (k[i] > best) {
          best = k[i];
          bi = i;
        }
      }
    }
  }
  return my_id;
}

// Largest of (v, i), the lower i among equals; i >= 0x7fffffff marks "none".
__device__ __forceinline__ void argmax64(double& v, int& i) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const double ov = __shfl_xor_sync(kFull, v, o);
    const int oi = __shfl_xor_sync(kFull, i, o);
    const bool none = i == 0x7fffffff, onone = oi == 0x7fffffff;
    if (!onone && (none || ov > v || (ov == v && oi < i))) {
      v = ov;
      i = oi;
    }
  }
}

// Exact choice value of a logit: s + bias.
__device__ __forceinline__ double choice64(float x, bool sigmoid, float m, double inv_z, float bias) {
  const double c = (x == kNegInf ? 0.0 : score64(x, sigmoid, m, inv_z)) + (double)bias;
  return c == c ? c : (double)kNegInf;
}

// Open groups by exact scores (rows whose fp32 group scores lie too close). g1, g2: the fp32 best
// values of group `lane` (choice values; without a bias the logits, which are exact). With a bias only
// the values that may be a group's best (two) within the error are computed exactly.
template <int EPL>
__device__ __noinline__ unsigned open_groups64(const float (&x)[EPL], const float (&c)[EPL], float g1, float g2,
                                               float tol, const float* bias, bool sigmoid, float m, double inv_z,
                                               const Shape& sh, int lane, double* buf) {
  const bool two = sh.top2 && sh.gsize > 1;
  double a = g1, b = g2;
  if (bias == nullptr) {
    a = choice64(g1, sigmoid, m, inv_z, 0.f);
    b = choice64(g2, sigmoid, m, inv_z, 0.f);
  } else {
    const float least = (two ? g2 : g1) - tol * (1.f + fabsf(two ? g2 : g1));
    double v[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane * EPL + i;
      const float t = __shfl_sync(kFull, least, min(e / sh.gsize, 31));
      v[i] = (double)kNegInf;
      if (e < sh.E && !(c[i] < t)) v[i] = choice64(x[i], sigmoid, m, inv_z, bias[e]);
    }
    group_top2<EPL, double>(v, sh, lane, buf, a, b);
  }
  uint32_t hi = 0u, lo = 0u;
  const double g = two ? a + b : a;
  if (lane < sh.groups) ord64(g == g ? g : (double)kNegInf, hi, lo);
  unsigned open;
  pick_list<true>(hi, lo, sh.top_groups, lane, open);
  return open;
}

// The K best experts by exact choice values among those of `live` (bit i: expert lane * EPL + i).
template <int EPL>
__device__ __noinline__ int pick_all64(const float (&x)[EPL], const float* bias, bool sigmoid, float m, double inv_z,
                                       unsigned live, int K, int lane) {
  double c[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    c[i] = (live >> i) & 1u ? choice64(x[i], sigmoid, m, inv_z, bias[lane * EPL + i]) : 0.0;
  int my_id = 0;
  for (int kk = 0; kk < K; ++kk) {
    double v = 0.0;
    int id = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (((live >> i) & 1u) && (id == 0x7fffffff || c[i] > v)) {
        v = c[i];
        id = lane * EPL + i;
      }
    argmax64(v, id);
    if (lane == kk) my_id = id;
    if (id / EPL == lane) live &= ~(1u << (id % EPL));
  }
  return my_id;
}

template <int EPL, bool F32>
__global__ void __launch_bounds__(kWarps * 32) route_scored_kernel(const RouteScoredParams p, const Shape sh, int vec, int vecb) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint2 cand[kWarps][32];
  extern __shared__ double dynbuf[];  // per warp E doubles (only when a group starts inside a lane)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x * kWarps + warp;
  if (t >= p.T) return;
  double* buf = dynbuf + (sh.lanes > 0 ? 0 : warp * sh.E);
  const int E = sh.E;
  const size_t row = (size_t)t * p.ld;
  const float* lf = reinterpret_cast<const float*>(p.logits) + row;
  const __nv_bfloat16* lh = reinterpret_cast<const __nv_bfloat16*>(p.logits) + row;
  float x[EPL];
  if (!F32 && EPL % 8 == 0 && vec && (lane + 1) * EPL <= E) {
#pragma unroll
    for (int i = 0; i < EPL / 8; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(lh + lane * EPL)[i];
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[i * 8 + 2 * j] = clean(__uint_as_float(w[j] << 16));
        x[i * 8 + 2 * j + 1] = clean(__uint_as_float(w[j] & 0xffff0000u));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane * EPL + i;
      x[i] = e < E ? clean(F32 ? lf[e] : __bfloat162float(lh[e])) : kNegInf;
    }
  }
  const bool sigm = p.sigmoid;
  float m = 0.f, z = 1.f;
  const bool need_z = !sigm && !p.renorm;  // (the weights' denominator)
  if (!sigm) {
    m = kNegInf;
#pragma unroll
    for (int i = 0; i < EPL; ++i) m = fmaxf(m, x[i]);
    m = unord32(__reduce_max_sync(kFull, ord32(m)));
    if (need_z) {
      z = 0.f;
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (x[i] > kNegInf) z += x[i] == m ? 1.f : expf(x[i] - m);
#pragma unroll
      for (int o = 16; o; o >>= 1) z += __shfl_xor_sync(kFull, z, o);
    }
  }
  double inv_z64 = 1.0;  // exact softmax denominator: needed where scores meet a bias
  if (!sigm && p.bias != nullptr) {
    double z64 = 0.0;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (x[i] > kNegInf) z64 += x[i] == m ? 1.0 : exp((double)x[i] - (double)m);
#pragma unroll
    for (int o = 16; o; o >>= 1) z64 += __shfl_xor_sync(kFull, z64, o);
    inv_z64 = z64 > 0.0 ? 1.0 / z64 : 0.0;
  }
  // fp32 choice values. A score (absolute value <= 1) is off by less than 2.5e-7 (argument rounded by
  // 2^-24 of itself, exponential 2 ulp, reciprocal 1 ulp: times s (1 - s)), adding the bias rounds by 2^-24
  // of the sum. Two values that are compared are off by less than 5e-7 + 1.2e-7 |c| together, within the
  // margin of kTol (1 + |c|) of a list. A group's sum of two is off by 5e-7 + 2^-24 (|c1| + |c2| + |sum|), and
  // its distance to the error's ends rounds by 2^-24 |sum| more: less than kSumErr + kSumRel (|c1| + |c2|).
  // (The operands count, not the sum: biases of opposite signs cancel in it, their roundings do not.)
  constexpr float kTol = 1e-6f, kSumErr = 5e-7f, kSumRel = 2e-7f;
  float c[EPL];
  if (p.bias == nullptr) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) c[i] = x[i];
  } else {
    const float inv_z = (float)inv_z64;
    float b[EPL];
    if (EPL % 4 == 0 && vecb && (lane + 1) * EPL <= E) {
#pragma unroll
      for (int i = 0; i < EPL / 4; ++i) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p.bias + lane * EPL) + i);
        b[4 * i] = v.x;
        b[4 * i + 1] = v.y;
        b[4 * i + 2] = v.z;
        b[4 * i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i) b[i] = lane * EPL + i < E ? __ldg(p.bias + lane * EPL + i) : kNegInf;
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      c[i] = clean((sigm ? sigmoid_fast(x[i]) : (x[i] == m ? 1.f : exp_fast(x[i] - m)) * inv_z) + b[i]);
  }
  unsigned open = kFull;
  if (sh.groups > 1) {
    float g1, g2, g, err = -1.f;
    group_top2<EPL, float>(c, sh, lane, reinterpret_cast<float*>(buf), g1, g2);
    g = g1;
    if (sh.top2 && sh.gsize > 1) {
      float s1 = g1, s2 = g2;
      if (p.bias == nullptr) {
        s1 = g1 == kNegInf ? 0.f : sigm ? sigmoid_fast(g1) : (g1 == m ? 1.f : exp_fast(g1 - m));
        s2 = g2 == kNegInf ? 0.f : sigm ? sigmoid_fast(g2) : (g2 == m ? 1.f : exp_fast(g2 - m));
      }
      g = clean(s1 + s2);
      // (an infinite value makes an infinite sum, which is exact)
      err = s1 < INFINITY && s2 > kNegInf ? kSumErr + kSumRel * (fabsf(s1) + fabsf(s2)) : 0.f;
    } else if (p.bias != nullptr) {
      err = fabsf(g) < INFINITY ? kSumErr + kSumRel * fabsf(g) : 0.f;
    }
    bool sure;
    open = open_groups32(g, sh, lane, err, sure);
    if (!sure) open = open_groups64<EPL>(x, c, g1, g2, kTol, p.bias, sigm, m, inv_z64, sh, lane, buf);
  }
  uint32_t k[EPL];
  unsigned live = 0;
  if (sh.lanes > 0) {  // the lane's experts are of one group
    const bool in = (open >> (lane / sh.lanes)) & 1u;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      k[i] = in && lane * EPL + i < E ? ord32(c[i]) : 0u;
      live |= (k[i] != 0u ? 1u : 0u) << i;
    }
  } else {
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane * EPL + i;
      k[i] = e < E && ((open >> (e / sh.gsize)) & 1u) ? ord32(c[i]) : 0u;
      live |= (k[i] != 0u ? 1u : 0u) << i;
    }
  }
  int my_id, listed = 33;
  uint2 my;
  float xi = kNegInf, si = -1.f;  // pick `lane`: its logit, its score where it is at hand
  if (sh.K <= kListK) listed = short_list<EPL>(k, sh.K, p.bias == nullptr ? 0.f : kTol, lane, cand[warp], my);
  if (listed <= 32) {
    unsigned taken;
    float xv = unord32(my.x), sv = 0.f;
    int src;
    if (p.bias == nullptr) {
      src = pick_list<false>(my.x, 0u, sh.K, lane, taken);
    } else {
      uint32_t hi = 0u, lo = 0u;
      if (lane < listed) {
        xv = clean(F32 ? lf[my.y] : __bfloat162float(lh[my.y]));
        const double s64 = xv == kNegInf ? 0.0 : score64(xv, sigm, m, inv_z64), v = s64 + (double)__ldg(p.bias + my.y);
        ord64(v == v ? v : (double)kNegInf, hi, lo);
        sv = (float)s64;
      }
      src = pick_list<true>(hi, lo, sh.K, lane, taken);
      if (sigm) si = __shfl_sync(kFull, sv, src);
    }
    my_id = __shfl_sync(kFull, (int)my.y, src);
    xi = __shfl_sync(kFull, xv, src);
  } else {
    my_id = p.bias == nullptr ? pick_all<EPL>(k, sh.K, lane)
                              : pick_all64<EPL>(x, p.bias, sigm, m, inv_z64, live, sh.K, lane);
    if (lane < sh.K) xi = clean(F32 ? lf[my_id] : __bfloat162float(lh[my_id]));
  }
  // weights: lane k takes pick k, in fp32 with the accurate exponential and divide
  const bool on = lane < sh.K;
  if (!on) xi = kNegInf;
  float s = 0.f;
  if (sigm) {
    if (on) {
      const float ex = expf(-fabsf(xi));
      s = si >= 0.f ? si : (xi >= 0.f ? 1.f : ex) / (1.f + ex);
    }
    if (p.renorm) {  // far below 0 a sigmoid is the exponential: relative to the largest it does not underflow
      const float mm = unord32(__reduce_max_sync(kFull, ord32(xi)));
      if (mm < -30.f) s = xi > kNegInf ? expf(xi - mm) : 0.f;
    }
  } else {
    // renormalised: relative to the largest pick, the softmax denominator cancels (next to an
    // infinite logit every other score is 0)
    float mm = m;
    if (p.renorm && m < INFINITY) mm = unord32(__reduce_max_sync(kFull, ord32(xi)));
    if (xi > kNegInf) s = xi == mm ? 1.f : expf(xi - mm);
    if (!p.renorm) s = z > 0.f ? s / z : 0.f;
  }
  if (p.renorm) {
    float sum = s;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    s = sum > 0.f ? s / sum : 0.f;
  }
  if (on) {
    p.ids[(size_t)t * sh.K + lane] = my_id;
    p.w[(size_t)t * sh.K + lane] = s * p.scale;
  }
}

template <int EPL>
cudaError_t launch_epl(const RouteScoredParams& p, const Shape& sh, int vec, int vecb, cudaStream_t s) {
  const dim3 grid((p.T + kWarps - 1) / kWarps);
  const size_t smem = sh.lanes > 0 ? 0 : (size_t)kWarps * sh.E * sizeof(double);
  if (p.f32) SQ_LAUNCH((route_scored_kernel<EPL, true>), grid, dim3(kWarps * 32), smem, s, 1, p, sh, vec, vecb);
  else SQ_LAUNCH((route_scored_kernel<EPL, false>), grid, dim3(kWarps * 32), smem, s, 1, p, sh, vec, vecb);
  return cudaGetLastError();
}

}  // namespace

cudaError_t moe_route_scored_launch(const RouteScoredParams& p, cudaStream_t s) {
  if (p.T == 0) return cudaSuccess;
  if (p.E < 1 || p.E > kRouteMaxExperts || p.groups < 1 || p.groups > kRouteMaxGroups || p.E % p.groups ||
      p.top_groups < 1 || p.top_groups > p.groups || p.K < 1 || p.K > kRouteMaxK ||
      p.K > p.E / p.groups * p.top_groups)
    return cudaErrorInvalidValue;
  Shape sh{p.E, p.K, p.groups, p.top_groups, p.E / p.groups, 0, p.top2};
  // experts per lane: the fewest that hold the row, preferring a count that divides the group so
  // that groups are whole lanes (their two best then meet by shuffles, not through shared memory)
  static const int kEpl[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16};
  int epl = 0;
  for (int c : kEpl)
    if (c * 32 >= p.E && (p.groups == 1 || sh.gsize % c == 0)) {
      epl = c;
      break;
    }
  if (epl) sh.lanes = p.groups == 1 ? 32 : sh.gsize / epl;
  for (int c : kEpl)
    if (!epl && c * 32 >= p.E) epl = c;
  const int vec = !p.f32 && p.ld % 8 == 0 && reinterpret_cast<uintptr_t>(p.logits) % 16 == 0;
  const int vecb = p.bias != nullptr && reinterpret_cast<uintptr_t>(p.bias) % 16 == 0;
  switch (epl) {
    case 1: return launch_epl<1>(p, sh, vec, vecb, s);
    case 2: return launch_epl<2>(p, sh, vec, vecb, s);
    case 3: return launch_epl<3>(p, sh, vec, vecb, s);
    case 4: return launch_epl<4>(p, sh, vec, vecb, s);
    case 5: return launch_epl<5>(p, sh, vec, vecb, s);
    case 6: return launch_epl<6>(p, sh, vec, vecb, s);
    case 8: return launch_epl<8>(p, sh, vec, vecb, s);
    case 10: return launch_epl<10>(p, sh, vec, vecb, s);
    case 12: return launch_epl<12>(p, sh, vec, vecb, s);
    default: return launch_epl<16>(p, sh, vec, vecb, s);
  }
}

}  // namespace sq
