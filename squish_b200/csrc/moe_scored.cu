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
// monotone in them): no rounding can reorder it. With a bias, or sums of two scores, c is compared
// in fp32 with a known error bound; a row in which two compared values lie closer than twice the
// bound is chosen again in fp64 by the same warp, so the ids are those of the exact scores.
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
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
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

// The two largest of (a1 >= a2) and (b1 >= b2).
template <class S>
__device__ __forceinline__ void merge2(S& a1, S& a2, S b1, S b2) {
  const S lo = a1 < b1 ? a1 : b1, hi = a1 < b1 ? b1 : a1;
  const S s2 = a2 < b2 ? b2 : a2;
  a1 = hi;
  a2 = lo < s2 ? s2 : lo;
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
    for (int i = 0; i < EPL; ++i) merge2(t1, t2, v[i], ninf);
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

// fp32 choice. gscore: this lane's group score (lane < groups); c: choice values. Returns false
// when two compared values lie within `tol` of each other (tol_g for groups; < 0: exact values).
template <int EPL>
__device__ __forceinline__ bool choose32(const float (&c)[EPL], float gscore, const Shape& sh, int lane, float tol_g,
                                         float tol, int& my_id) {
  bool sure = true;
  unsigned open = kFull;
  if (sh.groups > 1) {
    uint32_t gk = lane < sh.groups ? ord32(clean(gscore)) : 0u;
    open = 0;
    float last = 0.f;
    for (int g = 0; g < sh.top_groups; ++g) {
      const uint32_t m = __reduce_max_sync(kFull, gk);
      const int win = __ffs(__ballot_sync(kFull, gk == m)) - 1;
      open |= 1u << win;
      if (lane == win) gk = 0u;
      last = unord32(m);
    }
    if (tol_g >= 0.f && sh.top_groups < sh.groups) {
      const float next = unord32(__reduce_max_sync(kFull, gk));
      if (!(last - next > tol_g * (1.f + fabsf(last)))) sure = false;
    }
  }
  uint32_t k[EPL];
  uint32_t best = 0u;
  int bi = 0;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane * EPL + i;
    bool in = e < sh.E;
    if (sh.groups > 1 && in) in = (open >> (sh.lanes > 0 ? lane / sh.lanes : e / sh.gsize)) & 1u;
    k[i] = in ? ord32(c[i]) : 0u;
    if (k[i] > best) {
      best = k[i];
      bi = i;
    }
  }
  my_id = 0;
  float prev = INFINITY;
  for (int kk = 0; kk < sh.K; ++kk) {
    const uint32_t m = __reduce_max_sync(kFull, best);
    const int win = __ffs(__ballot_sync(kFull, best == m)) - 1;
    const int id = win * EPL + __shfl_sync(kFull, bi, win);
    if (lane == kk) my_id = id;
    if (tol >= 0.f) {
      const float v = unord32(m);
      if (kk > 0 && !(prev - v > tol * (1.f + fabsf(v)))) sure = false;
      prev = v;
    }
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
  if (tol >= 0.f) {  // the first value left out
    const uint32_t m = __reduce_max_sync(kFull, best);
    if (m != 0u && !(prev - unord32(m) > tol * (1.f + fabsf(prev)))) sure = false;
  }
  return sure;
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

// The same choice in fp64, from the logits (rows whose fp32 values lie too close): by s + bias, or,
// without a bias, by the logits, with only the groups ranked by sums of scores.
template <int EPL>
__device__ __noinline__ int choose64(const float (&x)[EPL], const float* bias, bool sigmoid, const Shape& sh, int lane,
                                     double* buf) {
  float m = kNegInf;
  double inv_z = 1.0;
  if (!sigmoid) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) m = fmaxf(m, x[i]);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
    double z = 0.0;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (x[i] > kNegInf) z += x[i] == m ? 1.0 : exp((double)x[i] - (double)m);
#pragma unroll
    for (int o = 16; o; o >>= 1) z += __shfl_xor_sync(kFull, z, o);
    inv_z = z > 0.0 ? 1.0 / z : 0.0;
  }
  double c[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane * EPL + i;
    c[i] = x[i];
    if (bias != nullptr)
      c[i] = e < sh.E ? (x[i] == kNegInf ? 0.0 : score64(x[i], sigmoid, m, inv_z)) + (double)bias[e] : (double)kNegInf;
    if (!(c[i] == c[i])) c[i] = (double)kNegInf;
  }
  unsigned open = kFull;
  if (sh.groups > 1) {
    double g1, g2;
    group_top2<EPL, double>(c, sh, lane, buf, g1, g2);
    double g = g1;
    if (sh.top2 && sh.gsize > 1) {
      if (bias == nullptr) {
        g1 = g1 == (double)kNegInf ? 0.0 : score64((float)g1, sigmoid, m, inv_z);
        g2 = g2 == (double)kNegInf ? 0.0 : score64((float)g2, sigmoid, m, inv_z);
      }
      g = g1 + g2;
    }
    bool taken = lane >= sh.groups;
    open = 0;
    for (int t = 0; t < sh.top_groups; ++t) {
      double v = g;
      int i = taken ? 0x7fffffff : lane;
      argmax64(v, i);
      open |= 1u << i;
      if (lane == i) taken = true;
    }
  }
  unsigned live = 0;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane * EPL + i;
    bool in = e < sh.E;
    if (sh.groups > 1 && in) in = (open >> (e / sh.gsize)) & 1u;
    if (in) live |= 1u << i;
  }
  int my_id = 0;
  for (int kk = 0; kk < sh.K; ++kk) {
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
__global__ void __launch_bounds__(kWarps * 32) route_scored_kernel(const RouteScoredParams p, const Shape sh, int vec) {
  pdl_wait();
  pdl_trigger();
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
  const bool need_z = !sigm && (p.bias != nullptr || !p.renorm);
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
  const float inv_z = z > 0.f ? 1.f / z : 0.f;
  // Error of the fp32 choice values: a score (absolute value <= 1) is off by less than 4e-7 (fast
  // exponential and divide), adding the bias rounds by 2^-24 of the sum; so 1e-6 (1 + |c|) covers a
  // difference of two, and twice that a difference of two sums of two.
  int my_id;
  bool sure;
  if (p.bias == nullptr) {
    float g = 0.f, tol_g = -1.f;
    if (sh.groups > 1) {
      float g1, g2;
      group_top2<EPL, float>(x, sh, lane, reinterpret_cast<float*>(buf), g1, g2);
      g = g1;
      if (sh.top2 && sh.gsize > 1) {
        auto sc = [&](float v) {
          if (v == kNegInf) return 0.f;
          return sigm ? __fdividef(1.f, 1.f + __expf(-v)) : (v == m ? 1.f : __expf(v - m));
        };
        g = sc(g1) + sc(g2);
        tol_g = 2e-6f;
      }
    }
    sure = choose32<EPL>(x, g, sh, lane, tol_g, -1.f, my_id);
  } else {
    float c[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane * EPL + i;
      float s = 0.f;
      if (x[i] > kNegInf) s = sigm ? __fdividef(1.f, 1.f + __expf(-x[i])) : (x[i] == m ? 1.f : __expf(x[i] - m)) * inv_z;
      c[i] = e < E ? clean(s + __ldg(p.bias + e)) : kNegInf;
    }
    float g = 0.f;
    if (sh.groups > 1) {
      float g1, g2;
      group_top2<EPL, float>(c, sh, lane, reinterpret_cast<float*>(buf), g1, g2);
      g = sh.top2 && sh.gsize > 1 ? g1 + g2 : g1;
    }
    sure = choose32<EPL>(c, g, sh, lane, 2e-6f, 1e-6f, my_id);
  }
  if (!sure) my_id = choose64<EPL>(x, p.bias, sigm, sh, lane, buf);
  // weights: lane k takes pick k, in fp32 with the accurate exponential and divide
  const bool on = lane < sh.K;
  const float xi = on ? clean(F32 ? lf[my_id] : __bfloat162float(lh[my_id])) : kNegInf;
  float s = 0.f;
  if (sigm) {
    if (on) {
      const float ex = expf(-fabsf(xi));
      s = (xi >= 0.f ? 1.f : ex) / (1.f + ex);
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
cudaError_t launch_epl(const RouteScoredParams& p, const Shape& sh, int vec, cudaStream_t s) {
  const dim3 grid((p.T + kWarps - 1) / kWarps);
  const size_t smem = sh.lanes > 0 ? 0 : (size_t)kWarps * sh.E * sizeof(double);
  if (p.f32) SQ_LAUNCH((route_scored_kernel<EPL, true>), grid, dim3(kWarps * 32), smem, s, 1, p, sh, vec);
  else SQ_LAUNCH((route_scored_kernel<EPL, false>), grid, dim3(kWarps * 32), smem, s, 1, p, sh, vec);
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
  switch (epl) {
    case 1: return launch_epl<1>(p, sh, vec, s);
    case 2: return launch_epl<2>(p, sh, vec, s);
    case 3: return launch_epl<3>(p, sh, vec, s);
    case 4: return launch_epl<4>(p, sh, vec, s);
    case 5: return launch_epl<5>(p, sh, vec, s);
    case 6: return launch_epl<6>(p, sh, vec, s);
    case 8: return launch_epl<8>(p, sh, vec, s);
    case 10: return launch_epl<10>(p, sh, vec, s);
    case 12: return launch_epl<12>(p, sh, vec, s);
    default: return launch_epl<16>(p, sh, vec, s);
  }
}

}  // namespace sq
