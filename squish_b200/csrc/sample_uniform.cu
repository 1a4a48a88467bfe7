// sample_uniform.cu — one token per row from a given uniform number u, by inverse transform.
//
// Order the tokens by logit, largest first, the lower index first among equals. With weights
// w = exp((l - max) / T) keep the prefix that min-p (w >= min_p), top-k (k tokens) and top-p (the
// shortest prefix whose mass reaches top_p of the mass of all tokens) allow, at least one token, and
// return the first token whose inclusive kept mass exceeds u * (kept mass). A disallowed (grammar
// mask), NaN or -inf logit is no token; a row without tokens returns -1. T <= 0 returns the first
// largest logit.
//
// A row of bf16 logits has few distinct values, and all of the above depends on the tokens only
// through (value, count) until the very last step. So a row is one histogram of its 16-bit keys in
// shared memory, one exponential (fp64) per distinct value instead of one per token, prefix sums over
// the bins, and a second pass that finds the n-th occurrence of the drawn value. No sort, and every
// comparison against a mass border is made in fp64: the token is the one the formula gives.
//
// The bins hold the values of magnitude [2^-31, 2^33) and zero: 16385 counters, 64 KB, so that
// three rows share an SM. A row with a value outside (none comes out of a model, but the format
// allows it) is counted again in four windows of the whole key space.
//
// A cluster of C CTAs shares a row when there are few rows: each counts a slice, owns 1/C of the
// bins (summed over the peers' shared memory) and the totals are exchanged through shared memory.
#include <cooperative_groups.h>

#include "kernels.h"
#include "launch.cuh"
#include "step_ops.h"

namespace cg = cooperative_groups;

namespace sq {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 16385;     // 8192 positive, zero, 8192 negative
constexpr int kMagLo = 0x3000;   // 2^-31
constexpr int kMagN = 0x2000;    // .. 2^33
constexpr int kWindow = 16384;   // bins of a window of the whole key space (four windows)
constexpr int kNone = 0x7fffffff;
constexpr int kHist = 33 * kThreads;  // counters, padded so that every thread's bins exist (C = 1: 33 each)
static_assert(kHist >= kBins && kHist % 4 == 0, "histogram size");

struct Shared {
  double mass[kWarps];
  int cnt[kWarps];
  int imin[kWarps];
  // exchanged between the CTAs of a row
  int first;       // first non-empty bin
  int odd;         // a value outside the main bins was seen
  double x_mass;   // mass of the CTA's bins
  int x_cnt;
  double x_kept;
  int x_sel;       // selecting thread of the row, -1
  int r_bits, r_rank;
  double r_z;
  int x_hits;
  unsigned long long best;  // greedy: (key, ~index)
  int whits[kWarps];
};

__device__ __forceinline__ double bf16_value(int bits) { return (double)__uint_as_float((unsigned)bits << 16); }

// bf16 bits of bin j: the main bins (win < 0) or window `win`, both in descending order of value
__device__ __forceinline__ int bin_bits(int j, int win) {
  if (win < 0) {
    if (j < kMagN) return kMagLo + kMagN - 1 - j;
    return j == kMagN ? 0 : (0x8000 | (kMagLo + (j - kMagN - 1)));
  }
  const int key = 0xffff - (win * kWindow + j);
  return (key & 0x8000) ? (key ^ 0x8000) : (~key & 0xffff);
}

// Count one value into the bins. Returns false for a value outside the main bins.
__device__ __forceinline__ bool count_bits(unsigned bits, int win, int* hist) {
  const unsigned mag = bits & 0x7fffu;
  if (win < 0) {
    const unsigned t = mag - (unsigned)kMagLo;
    if (t < (unsigned)kMagN) {
      atomicAdd(hist + ((bits & 0x8000u) ? kMagN + 1 + (int)t : kMagN - 1 - (int)t), 1);
      return true;
    }
    if (mag == 0) {
      atomicAdd(hist + kMagN, 1);
      return true;
    }
    return mag > 0x7f80u || bits == 0xff80u;  // NaN and -inf are no tokens; anything else is outside
  }
  if (mag > 0x7f80u || bits == 0xff80u) return true;
  const unsigned b = mag == 0 ? 0u : bits;
  const unsigned o = 0xffffu - ((b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u));
  if ((int)(o >> 14) == win) atomicAdd(hist + (o & (kWindow - 1)), 1);
  return true;
}

// A row slice: `head` single values, then 16-byte groups of 8, then `tail` single values.
struct Slice {
  const __nv_bfloat16* row;
  const uint32_t* mask;
  int i0, head;      // first index, single values before the groups
  int v0, nv;        // index of the first group's first value, groups
  int t0, tail;

  __device__ __forceinline__ unsigned allowed(int i) const {
    return mask == nullptr ? 1u : (mask[i >> 5] >> (i & 31)) & 1u;
  }
  __device__ __forceinline__ unsigned allowed8(int i) const {
    if (mask == nullptr) return 0xffu;
    const int s = i & 31;
    unsigned w = mask[i >> 5] >> s;
    if (s > 24) w |= mask[(i >> 5) + 1] << (32 - s);
    return w & 0xffu;
  }
  __device__ __forceinline__ unsigned bits(int i) const {
    return *reinterpret_cast<const unsigned short*>(row + i);
  }
  __device__ __forceinline__ uint4 group(int g) const { return *reinterpret_cast<const uint4*>(row + v0 + 8 * g); }
};

__device__ __forceinline__ Slice make_slice(const SampleUniformParams& p, int row, int rank, int C) {
  Slice s;
  s.row = p.logits + (size_t)row * p.ld;
  s.mask = p.allow_mask ? p.allow_mask + (size_t)row * ((p.V + 31) / 32) : nullptr;
  const int lead = (int)((16 - (reinterpret_cast<uintptr_t>(s.row) & 15)) & 15) / 2;  // values up to a 16-byte border
  const int a = lead < p.V ? lead : p.V;
  const int groups = (p.V - a) / 8;
  const int g0 = (int)((long long)groups * rank / C), g1 = (int)((long long)groups * (rank + 1) / C);
  s.i0 = 0;
  s.head = rank == 0 ? a : 0;
  s.v0 = a + 8 * g0;
  s.nv = g1 - g0;
  s.t0 = a + 8 * groups;
  s.tail = rank == C - 1 ? p.V - s.t0 : 0;
  return s;
}

template <int C>
__device__ __forceinline__ void row_sync(cg::cluster_group& cl) {
  if constexpr (C == 1) __syncthreads();
  else cl.sync();
}

template <int C>
__global__ void __launch_bounds__(kThreads, 2) sample_uniform_kernel(const SampleUniformParams p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(16) int hist[];
  __shared__ Shared sh;
  cg::cluster_group cl = cg::this_cluster();
  const int row = blockIdx.x;
  const int rank = C == 1 ? 0 : (int)blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto peer = [&](int r) -> Shared* {
    if constexpr (C == 1) return &sh;
    else return cl.map_shared_rank(&sh, r);
  };
  const Slice sl = make_slice(p, row, rank, C);
  const float tf = p.temperature ? p.temperature[row] : 0.f;

  if (!(tf > 0.f)) {  // greedy: largest key, lowest index
    unsigned long long best = 0;
    auto take = [&](unsigned b, int i) {
      if ((b & 0x7fffu) > 0x7f80u || b == 0xff80u) return;
      if ((b & 0x7fffu) == 0) b = 0;
      const unsigned key = (b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u);
      const unsigned long long v = ((unsigned long long)key << 32) | (unsigned)(~i);
      best = v > best ? v : best;
    };
    if (tid < sl.head && sl.allowed(sl.i0 + tid)) take(sl.bits(sl.i0 + tid), sl.i0 + tid);
    if (tid < sl.tail && sl.allowed(sl.t0 + tid)) take(sl.bits(sl.t0 + tid), sl.t0 + tid);
    for (int g = tid; g < sl.nv; g += kThreads) {
      const uint4 v = sl.group(g);
      const unsigned w[4] = {v.x, v.y, v.z, v.w};
      const int i = sl.v0 + 8 * g;
      const unsigned ok = sl.allowed8(i);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if ((ok >> j) & 1u) take((w[j >> 1] >> (16 * (j & 1))) & 0xffffu, i + j);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const unsigned long long v = __shfl_xor_sync(0xffffffffu, best, o);
      best = v > best ? v : best;
    }
    if (tid == 0) sh.best = 0;
    __syncthreads();
    if (lane == 0) atomicMax(&sh.best, best);
    row_sync<C>(cl);
    if (rank == 0 && tid == 0) {
      best = 0;
      for (int r = 0; r < C; ++r) best = max(best, peer(r)->best);
      p.out_tokens[row] = best ? (int)~(unsigned)best : -1;
      if (p.out_logprob) p.out_logprob[row] = best ? 0.f : -INFINITY;
    }
    if constexpr (C > 1) cl.sync();
    return;
  }

  const double inv_t = 1.0 / (double)tf;
  const double min_p = p.min_p ? (double)p.min_p[row] : 0.0;
  const double top_p = p.top_p ? (double)p.top_p[row] : 1.0;
  const int top_k = p.top_k ? p.top_k[row] : 0;
  const long long K = top_k > 0 ? top_k : (long long)kNone;

  if (tid == 0) {
    sh.odd = 0;
    sh.x_sel = -1;
  }
  constexpr int kPer = (kBins + C * kThreads - 1) / (C * kThreads);  // bins of a thread (of the cluster's C * 512)
  const int gtid = rank * kThreads + tid;
  const int j0 = gtid * kPer;
  // counts of bins [j0, j0 + kPer) over the whole row: the histogram itself, or its sums over the
  // peers (kPer is odd: threads stay on distinct banks)
  int* cnt = hist + (C == 1 ? tid * kPer : kHist + tid * kPer);

  // histogram of this CTA's slice, then the row's counts of the thread's own bins
  auto count_row = [&](int win) {
    for (int i = tid; i < kHist / 4; i += kThreads) reinterpret_cast<int4*>(hist)[i] = make_int4(0, 0, 0, 0);
    __syncthreads();
    bool inside = true;
    if (tid < sl.head && sl.allowed(sl.i0 + tid)) inside &= count_bits(sl.bits(sl.i0 + tid), win, hist);
    if (tid < sl.tail && sl.allowed(sl.t0 + tid)) inside &= count_bits(sl.bits(sl.t0 + tid), win, hist);
    for (int g = tid; g < sl.nv; g += kThreads) {
      const uint4 v = sl.group(g);
      const unsigned w[4] = {v.x, v.y, v.z, v.w};
      const unsigned ok = sl.allowed8(sl.v0 + 8 * g);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if ((ok >> j) & 1u) inside &= count_bits((w[j >> 1] >> (16 * (j & 1))) & 0xffffu, win, hist);
    }
    if (!inside) sh.odd = 1;
    row_sync<C>(cl);
    if constexpr (C > 1) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        int c = 0;
        if (j0 + i < kBins)
          for (int r = 0; r < C; ++r) c += cl.map_shared_rank(hist, r)[j0 + i];
        cnt[i] = c;
      }
    }
  };

  count_row(-1);
  bool odd = false;
  for (int r = 0; r < C; ++r) odd |= peer(r)->odd != 0;
  const int w_first = odd ? 0 : -1, w_end = odd ? 4 : 0;  // windows [w_first, w_end)

  // one window's counts in cnt[] (the main bins stay there from the first pass)
  auto open_window = [&](int win) {
    if (win < 0) return;
    row_sync<C>(cl);  // peers have read the previous window
    count_row(win);
  };

  // ---- largest value
  int vbits = -1;
  for (int win = w_first; win < w_end && vbits < 0; ++win) {
    open_window(win);
    int first = kNone;
#pragma unroll
    for (int i = kPer - 1; i >= 0; --i)
      if (cnt[i] > 0) first = j0 + i;
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) sh.imin[warp] = first;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kWarps; ++w) first = min(first, sh.imin[w]);
      sh.first = first;
    }
    row_sync<C>(cl);
    first = kNone;
    for (int r = 0; r < C; ++r) first = min(first, peer(r)->first);
    if (first != kNone) vbits = bin_bits(first, win);
    row_sync<C>(cl);
  }
  if (vbits < 0) {  // no token at all (the same in every CTA of the row)
    if (rank == 0 && tid == 0) {
      p.out_tokens[row] = -1;
      if (p.out_logprob) p.out_logprob[row] = -INFINITY;
    }
    if constexpr (C > 1) cl.sync();
    return;
  }
  const double vmax = bf16_value(vbits);
  auto logw = [&](int bits) -> double {
    const double v = bf16_value(bits);
    return v == vmax ? 0.0 : (v - vmax) * inv_t;
  };

  // Mass and count of the thread's bins, and of all bins before them (in this window).
  double mass = 0.0, m0 = 0.0, w_hi = 0.0, w_lo = 0.0;
  int n = 0;
  long long n0 = 0;
  double win_mass = 0.0;
  long long win_cnt = 0;
  auto prefix = [&](int win) {
    mass = 0.0;
    n = 0;
    w_hi = w_lo = 0.0;
#pragma unroll 1
    for (int i = 0; i < kPer; ++i) {
      const int c = cnt[i];
      if (c > 0) {
        const double w = exp(logw(bin_bits(j0 + i, win)));
        if (n == 0) w_hi = w;
        w_lo = w;
        n += c;
        mass += (double)c * w;
      }
    }
    double im = mass;
    int in = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double a = __shfl_up_sync(0xffffffffu, im, o);
      const int b = __shfl_up_sync(0xffffffffu, in, o);
      if (lane >= o) {
        im += a;
        in += b;
      }
    }
    double em = __shfl_up_sync(0xffffffffu, im, 1);
    int en = __shfl_up_sync(0xffffffffu, in, 1);
    if (lane == 0) {
      em = 0.0;
      en = 0;
    }
    __syncthreads();
    if (lane == 31) {
      sh.mass[warp] = im;
      sh.cnt[warp] = in;
    }
    __syncthreads();
    double tm = 0.0;
    int tn = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) {
        em += tm;
        en += tn;
      }
      tm += sh.mass[w];
      tn += sh.cnt[w];
    }
    if (tid == 0) {
      sh.x_mass = tm;
      sh.x_cnt = tn;
    }
    row_sync<C>(cl);
    win_mass = 0.0;
    win_cnt = 0;
    for (int r = 0; r < C; ++r) {
      if (r == rank) {
        em += win_mass;
        en += (int)win_cnt;
      }
      win_mass += peer(r)->x_mass;
      win_cnt += peer(r)->x_cnt;
    }
    m0 = em;
    n0 = en;
  };

  double z_all = 0.0;
  for (int win = w_first; win < w_end; ++win) {
    if (win >= 0) open_window(win);
    prefix(win);
    z_all += win_mass;
  }
  const double border = top_p < 1.0 ? top_p * z_all : INFINITY;

  // Tokens of bin (count c, weight w) that are kept, after bm mass and bn tokens before it.
  auto keep = [&](int c, double w, double bm, long long bn) -> int {
    if (bn == 0) {  // the first value: at least one token
      const int k = !(w >= min_p) ? 1 : c;
      long long t = min((long long)k, K);
      if (border < INFINITY) t = min(t, (long long)fmax(1.0, fmin((double)c, ceil((border - bm) / w))));
      return (int)t;
    }
    if (!(w >= min_p) || bn >= K || bm >= border) return 0;
    long long t = min((long long)c, K - bn);
    if (border < INFINITY && w > 0.0) t = min(t, (long long)fmax(1.0, fmin((double)c, ceil((border - bm) / w))));
    return (int)t;
  };
  // Walk the thread's bins: kept mass, and, for target >= 0, the kept bin that holds the target.
  auto walk = [&](int win, double bm, long long bn, double target, int* bits, int* rank_in) -> double {
    double kept = 0.0, m = bm;
    long long k0 = bn;
#pragma unroll 1
    for (int i = 0; i < kPer; ++i) {
      const int c = cnt[i];
      if (c <= 0) continue;
      const int b = bin_bits(j0 + i, win);
      const double w = exp(logw(b));
      const int t = keep(c, w, m, k0);
      if (t > 0 && bits != nullptr && (m <= target || *bits < 0)) {
        *bits = b;
        const double q = w > 0.0 ? floor((target - m) / w) : 0.0;
        *rank_in = (int)fmax(0.0, fmin(q, (double)(t - 1)));
      }
      kept += (double)t * w;
      m += (double)c * w;
      k0 += c;
      if (t < c) break;  // the kept tokens are a prefix
    }
    return kept;
  };

  // ---- kept mass
  double total = 0.0, base_m = 0.0;
  long long base_n = 0;
  double kept = 0.0;
  for (int win = w_first; win < w_end; ++win) {
    if (win >= 0) {
      open_window(win);
      prefix(win);
    }
    const double bm = base_m + m0;
    const long long bn = base_n + n0;
    kept = 0.0;
    if (n > 0) {
      if (bn > 0 && (bn >= K || bm >= border || !(w_hi >= min_p))) kept = 0.0;                   // past the end
      else if (bn > 0 && bn + n <= K && bm + mass < border && w_lo >= min_p) kept = mass;        // all inside
      else kept = walk(win, bm, bn, -1.0, nullptr, nullptr);
    }
    double s = kept;
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    __syncthreads();
    if (lane == 0) sh.mass[warp] = s;
    __syncthreads();
    if (tid == 0) {
      s = 0.0;
      for (int w = 0; w < kWarps; ++w) s += sh.mass[w];
      sh.x_kept = s;
    }
    row_sync<C>(cl);
    for (int r = 0; r < C; ++r) total += peer(r)->x_kept;
    base_m += win_mass;
    base_n += win_cnt;
    if constexpr (C > 1) {
      if (odd) cl.sync();
    } else {
      __syncthreads();
    }
  }

  // ---- the draw: the last kept bin whose preceding mass is <= target
  float u = p.uniforms[row];
  u = u > 0.f ? fminf(u, 1.f) : 0.f;
  const double target = (double)u * total;
  base_m = 0.0;
  base_n = 0;
  int bits = -1, nth = 0;
  for (int win = w_first; win < w_end; ++win) {
    if (win >= 0) {
      open_window(win);
      prefix(win);
    }
    const double bm = base_m + m0;
    const long long bn = base_n + n0;
    bool cand = false;
    if (n > 0 && (bn == 0 || (bm <= target && bn < K && bm < border && w_hi >= min_p))) cand = true;
    const int best = __reduce_max_sync(0xffffffffu, cand ? gtid : -1);
    __syncthreads();
    if (lane == 0) sh.imin[warp] = best;
    __syncthreads();
    if (tid == 0) {
      int b = -1;
      for (int w = 0; w < kWarps; ++w) b = max(b, sh.imin[w]);
      sh.x_sel = b;
    }
    row_sync<C>(cl);
    int sel = -1;
    for (int r = 0; r < C; ++r) sel = max(sel, peer(r)->x_sel);
    if (sel == gtid) {
      int b = -1, k = 0;
      walk(win, bm, bn, target, &b, &k);
      sh.r_bits = b;
      sh.r_rank = k;
    }
    row_sync<C>(cl);
    if (sel >= 0) {  // (a later window's candidate replaces an earlier one's)
      const Shared* o = peer(sel / kThreads);
      bits = o->r_bits;
      nth = o->r_rank;
    }
    base_m += win_mass;
    base_n += win_cnt;
  }

  // ---- the nth token (in index order) whose value is `bits`: each warp takes a contiguous part
  const int gper = (sl.nv + kWarps - 1) / kWarps;
  const int ga = min(sl.nv, warp * gper), gb = min(sl.nv, ga + gper);
  auto canon = [](unsigned b) -> int { return (b & 0x7fffu) == 0 ? 0 : (int)b; };
  auto match8 = [&](int g) -> unsigned {
    const uint4 v = sl.group(g);
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m |= (canon((w[j >> 1] >> (16 * (j & 1))) & 0xffffu) == bits ? 1u : 0u) << j;
    return m == 0 ? 0u : m & sl.allowed8(sl.v0 + 8 * g);
  };
  auto match1 = [&](int i) -> bool { return canon(sl.bits(i)) == bits && sl.allowed(i); };
  const unsigned hm = __ballot_sync(0xffffffffu, warp == 0 && lane < sl.head && match1(sl.i0 + lane));
  const unsigned tm = __ballot_sync(0xffffffffu, warp == kWarps - 1 && lane < sl.tail && match1(sl.t0 + lane));
  int hits = 0;
  for (int g = ga + lane; g < gb; g += 32) hits += __popc(match8(g));
  hits = __reduce_add_sync(0xffffffffu, hits) + __popc(hm) + __popc(tm);
  if (lane == 0) sh.whits[warp] = hits;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) before = all;
    all += sh.whits[w];
  }
  if (tid == 0) sh.x_hits = all;
  row_sync<C>(cl);
  for (int r = 0; r < rank; ++r) before += peer(r)->x_hits;
  const int want = nth - before;  // among this warp's tokens
  if (want >= 0 && want < hits) {
    int tok = -1;
    int seen = 0;
    if (want < __popc(hm)) {
      tok = sl.i0 + (__fns(hm, 0, want + 1));
    } else {
      seen = __popc(hm);
      for (int g = ga; g < gb && tok < 0; g += 32) {
        const unsigned m = g + lane < gb ? match8(g + lane) : 0u;
        int inc = __popc(m);
        const int own = inc;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += v;
        }
        const int need = want - seen;  // 0-based within this chunk
        int mine = -1;
        if (need >= inc - own && need < inc) mine = sl.v0 + 8 * (g + lane) + (int)__fns(m, 0, need - (inc - own) + 1);
        tok = __reduce_max_sync(0xffffffffu, mine);
        seen += __shfl_sync(0xffffffffu, inc, 31);
      }
      if (tok < 0) tok = sl.t0 + (int)__fns(tm, 0, want - seen + 1);
    }
    if (lane == 0) {
      p.out_tokens[row] = tok;
      if (p.out_logprob) p.out_logprob[row] = (float)(logw(bits) - log(total));
    }
  }
  if constexpr (C > 1) cl.sync();  // peers may still read this CTA's shared memory
}

template <int C>
cudaError_t launch_c(const SampleUniformParams& p, cudaStream_t s) {
  constexpr int per = (kBins + C * kThreads - 1) / (C * kThreads);
  constexpr size_t smem = (size_t)(kHist + (C > 1 ? per * kThreads : 0)) * sizeof(int);
  cudaError_t e = cudaFuncSetAttribute(sample_uniform_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  SQ_LAUNCH(sample_uniform_kernel<C>, dim3(p.B, 1, C), dim3(kThreads), smem, s, C, p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t sample_uniform_launch(const SampleUniformParams& p, int num_sms, cudaStream_t s) {
  if (p.B == 0) return cudaSuccess;
  if (p.V <= 0) return cudaErrorInvalidValue;
  // CTAs per row: as many as the SMs hold at one row each, at least 4096 values per CTA
  int c = 8;
  while (c > 1 && ((long long)p.B * c > 2 * num_sms || p.V / c < 4096)) c >>= 1;
  switch (c) {
    case 8: return launch_c<8>(p, s);
    case 4: return launch_c<4>(p, s);
    case 2: return launch_c<2>(p, s);
    default: return launch_c<1>(p, s);
  }
}

}  // namespace sq
