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
// The bins hold the values of magnitude [2^-31, 2^33) and zero: 16385 counters, 64 KB, so that rows
// share an SM. Two values of a 32-bit word become two byte offsets with three integer operations;
// a word with another value takes the checked path, and a row with a finite value outside (none
// comes out of a model, but the format allows it) is done by one CTA in four windows of the whole
// key space. Counting costs one shared-memory atomic per token (2 bytes of logits), and the row is
// loaded in 16-byte groups, four in flight per thread.
//
// A cluster of C CTAs shares a row when there are few rows: each counts a slice and owns 1/C of the
// bins (summed over the peers' shared memory); three exchanges through shared memory (masses, kept
// masses, the drawn value) make the draw, and a fourth keeps the memory alive.
//
// Measured (V 152064, temperature only): 1 row 16 us (a chain of five cluster exchanges and as many
// block sums in fp64, 27000 clocks), 64 rows 23 us, 256 rows 52 us (78 MB: 12 us at the copy rate). The
// atomics are 7 us of a row on its SM (4752 of its warps', 2.8 clocks each), 14 us for the two rows that
// share one; in the rest the warps wait, first of all for loads (256 rows with mixed filters and masks, 63
// us: an instruction issues in 42 % of the cycles, loads are the largest stall, then fixed latencies and
// barriers), with 256 rows on 148 SMs leaving 40 of them one row. With one exponential per token, serial walks
// over a thread's bins and counters read in the owner's order it was 34, 78 and 122 us.
#include <cooperative_groups.h>

#include "exp_neg.cuh"
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
constexpr int kSpare = kBins + 3;   // 32 spare counters, one per lane, for disallowed values
constexpr int kHist = kSpare + 32;  // counters, in whole 16-byte groups
static_assert(kHist % 4 == 0, "histogram size");

// i-th signed value in descending order -> bin (zero is bin kMagN)
__device__ __forceinline__ int nth_bin(int i) { return i + (i >= kMagN); }

struct Shared {
  double mass[2][kWarps];
  int cnt[kWarps];
  int imin[2][kWarps];
  int whits[2][kWarps];
  int odd;          // a value outside the main bins was seen
  // written by the CTAs of a row (each in every peer's memory, so that all reads are local)
  struct {
    double mass, kept;
    int first, cnt;  // first non-empty bin of the CTA's range, tokens
  } in[8];
  double scale[8];  // their masses on the row's scale
  int edge;  // thread at the end of the kept prefix (kThreads: none)
  // its entries and what precedes them, per warp
  struct {
    int first, n;
    long long n0;
    double m0;
  } end[kWarps];
  int r_bits, r_rank;
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
// Counter of a main value: the low 13 bits tell the magnitudes of the range apart, bit 13 the sign.
__device__ __forceinline__ int main_at(int bits) { return bits == 0 ? 2 * kMagN : (bits & 0x1fff) | ((bits & 0x8000) >> 2); }

// Count one value into the main bins. Returns false for a value outside.
__device__ __forceinline__ bool count_main(unsigned bits, int* hist) {
  const unsigned mag = bits & 0x7fffu;
  if (mag == 0) bits = 0;
  if (mag - (unsigned)kMagLo < (unsigned)kMagN || mag == 0) {
    atomicAdd(hist + main_at((int)bits), 1);
    return true;
  }
  return mag > 0x7f80u || bits == 0xff80u;  // NaN and -inf are no tokens; anything else is outside
}
// Count one value of window `win` of the whole key space.
__device__ __forceinline__ void count_window(unsigned bits, int win, int* hist) {
  const unsigned mag = bits & 0x7fffu;
  if (mag > 0x7f80u || bits == 0xff80u) return;
  if (mag == 0) bits = 0;
  const unsigned o = 0xffffu - ((bits & 0x8000u) ? (~bits & 0xffffu) : (bits | 0x8000u));
  if ((int)(o >> 14) == win) atomicAdd(hist + (o & (kWindow - 1)), 1);
}
// Both values of a word in the main bins?
__device__ __forceinline__ bool main_word(unsigned w) {
  return (((w & 0x7fff7fffu) + 0x50005000u) & 0xe000e000u) == 0x80008000u;  // magnitude >> 12 is 3 or 4
}
// Count both values of a word (ok: bit 0 / 1 set = the lower / upper value is allowed; others go to the
// lane's spare counter, which costs a select where a branch per value cost twice the row's time).
template <bool kAll>
__device__ __forceinline__ void count_word(unsigned w, unsigned ok, int* hist) {
  const unsigned o = (((w << 2) & 0x7ffc7ffcu) | (w & 0x80008000u));  // two byte offsets 4 * main_at
  const unsigned spare = 4u * (kSpare + (threadIdx.x & 31));
  char* h = reinterpret_cast<char*>(hist);
  atomicAdd(reinterpret_cast<int*>(h + (kAll || (ok & 1u) ? o & 0xffffu : spare)), 1);
  atomicAdd(reinterpret_cast<int*>(h + (kAll || (ok & 2u) ? o >> 16 : spare)), 1);
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
    // bits i .. i + 7: the word of i and that of i + 7 (the same, or the next one)
    return __funnelshift_r(mask[i >> 5], mask[(i + 7) >> 5], i & 31) & 0xffu;
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

__device__ __forceinline__ int canon(unsigned b) { return (b & 0x7fffu) == 0 ? 0 : (int)b; }

// Row-wide rules of the draw.
struct Rules {
  double inv_t, min_p, border;  // border: mass a top-p prefix has to reach (inf: off)
  long long K;
  double vmax;

  __device__ __forceinline__ double logw(int bits) const {
    const double v = bf16_value(bits);
    return v == vmax ? 0.0 : (v - vmax) * inv_t;
  }
  // Tokens kept of a value with c tokens of weight w, after bm mass and bn tokens before it.
  __device__ __forceinline__ int keep(int c, double w, double bm, long long bn) const {
    long long t = c;
    if (bn > 0) {
      if (!(w >= min_p) || bn >= K || bm >= border) return 0;
      t = min(t, K - bn);
    } else {  // the first value: at least one token
      if (!(w >= min_p)) t = 1;
      t = min(t, K);
    }
    if (border < INFINITY && (w > 0.0 || bn == 0))
      t = min(t, (long long)fmax(1.0, fmin((double)c, ceil((border - bm) / w))));
    return (int)t;
  }
};

// Kept mass of bins [j0, j0 + per) (counts through `at`), after bm mass and bn tokens; with `bits`,
// also the last kept value whose preceding mass is <= target, and the target's place among its tokens.
template <class At>
__device__ double walk(const Rules& rule, At at, int j0, int per, int win, double bm, long long bn, double target,
                       int* bits, int* place) {
  double kept = 0.0, m = bm;
  long long k0 = bn;
  for (int i = 0; i < per; ++i) {
    const int c = at(i);
    if (c <= 0) continue;
    const int b = bin_bits(j0 + i, win);
    const double w = exp_neg(rule.logw(b));
    const int t = rule.keep(c, w, m, k0);
    if (t > 0 && bits != nullptr && (m <= target || *bits < 0)) {
      *bits = b;
      *place = (int)fmax(0.0, fmin(w > 0.0 ? floor((target - m) / w) : 0.0, (double)(t - 1)));
    }
    kept += (double)t * w;
    m += (double)c * w;
    k0 += c;
    if (t < c) break;  // the kept tokens are a prefix
  }
  return kept;
}

// The same by a warp over entries [first, first + cnt) of a list of non-empty bins (entry -> bin), one
// entry per lane. All lanes return the kept mass; `bits` and `place` (when given) are set in all lanes.
template <class Bin, class Cnt>
__device__ double warp_walk(const Rules& rule, Bin bin, Cnt count, int first, int cnt, double bm, long long bn,
                            double target, int* bits, int* place) {
  const int lane = threadIdx.x & 31;
  double kept = 0.0;
  for (int e = 0; e < cnt; e += 32) {
    const bool on = e + lane < cnt;
    int b = 0, c = 0;
    double w = 0.0;
    if (on) {
      const int j = bin(first + e + lane);
      b = bin_bits(j, -1);
      c = count(j);
      w = exp_neg(rule.logw(b));
    }
    double im = (double)c * w;
    int in = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double a = __shfl_up_sync(0xffffffffu, im, o);
      const int d = __shfl_up_sync(0xffffffffu, in, o);
      if (lane >= o) {
        im += a;
        in += d;
      }
    }
    double m = __shfl_up_sync(0xffffffffu, im, 1);
    m = bm + (lane ? m : 0.0);
    const int t = on ? rule.keep(c, w, m, bn + in - c) : 0;
    double k = (double)t * w;
#pragma unroll
    for (int o = 16; o; o >>= 1) k += __shfl_xor_sync(0xffffffffu, k, o);
    kept += k;
    if (bits != nullptr) {
      unsigned hit = __ballot_sync(0xffffffffu, t > 0 && m <= target);
      if (hit == 0 && *bits < 0) hit = 1u;  // (rounding put the first start above the target)
      if (hit != 0) {
        const int src = 31 - __clz(hit);
        const int pl = (int)fmax(0.0, fmin(w > 0.0 ? floor((target - m) / w) : 0.0, (double)(t - 1)));
        *bits = __shfl_sync(0xffffffffu, b, src);
        *place = __shfl_sync(0xffffffffu, pl, src);
      }
    }
    bm += __shfl_sync(0xffffffffu, im, 31);
    bn += __shfl_sync(0xffffffffu, in, 31);
  }
  return kept;
}

// Exclusive prefix over the block of (mass, n), and the block's totals. These reductions take one
// barrier each; calls that follow one another alternate between two rows of `sh` (`turn`).
__device__ __forceinline__ void block_prefix(Shared& sh, int turn, double mass, int n, double& em, int& en, double& tm,
                                             int& tn) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
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
  em = __shfl_up_sync(0xffffffffu, im, 1);
  en = __shfl_up_sync(0xffffffffu, in, 1);
  if (lane == 0) {
    em = 0.0;
    en = 0;
  }
  if (lane == 31) {
    sh.mass[turn][warp] = im;
    sh.cnt[warp] = in;
  }
  __syncthreads();
  // the warps' sums: lane w takes warp w (fp64 additions one after another would be the longest wait here)
  static_assert(kWarps == 16, "one lane per warp sum");
  im = sh.mass[turn][lane & 15];
  in = sh.cnt[lane & 15];
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    const double a = __shfl_up_sync(0xffffffffu, im, o, 16);
    const int b = __shfl_up_sync(0xffffffffu, in, o, 16);
    if ((lane & 15) >= o) {
      im += a;
      in += b;
    }
  }
  tm = __shfl_sync(0xffffffffu, im, 15);
  tn = __shfl_sync(0xffffffffu, in, 15);
  const double bm = __shfl_sync(0xffffffffu, im, (warp + 15) & 15);
  const int bn = __shfl_sync(0xffffffffu, in, (warp + 15) & 15);
  if (warp > 0) {
    em += bm;
    en += bn;
  }
}
__device__ __forceinline__ int block_min(Shared& sh, int turn, int v) {
  v = __reduce_min_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) sh.imin[turn][threadIdx.x >> 5] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) v = min(v, sh.imin[turn][w]);
  return v;
}
__device__ __forceinline__ double block_sum(Shared& sh, int turn, double s) {
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sh.mass[turn][threadIdx.x >> 5] = s;
  __syncthreads();
  s = sh.mass[turn][threadIdx.x & 15];
#pragma unroll
  for (int o = 8; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// Index of the nth (from 0) set bit.
__device__ __forceinline__ int nth_bit(unsigned m, int n) {
  for (; n > 0; --n) m &= m - 1u;
  return __ffs(m) - 1;
}

// The nth token (in index order, from 0) of the slice whose value is `bits`, written to out_tokens[row].
// The block reads the slice in rounds of 4096 groups, each warp 256 consecutive ones, and stops with the
// round that holds the token.
__device__ __forceinline__ void find_token(const SampleUniformParams& p, int row, const Slice& sl, Shared& sh, int bits,
                                           int nth) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned pat = (unsigned)bits * 0x10001u;
  auto match8 = [&](const uint4& v, int g) -> unsigned {
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
    if (bits != 0) {  // no half-word of w ^ pat is zero: (x - 1) & ~x has no sign bit (it may have one without)
      unsigned any = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned x = w[j] ^ pat;
        any |= (x - 0x00010001u) & ~x;
      }
      if ((any & 0x80008000u) == 0) return 0u;
    }
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m |= (canon((w[j >> 1] >> (16 * (j & 1))) & 0xffffu) == bits ? 1u : 0u) << j;
    return m == 0 ? 0u : m & sl.allowed8(sl.v0 + 8 * g);
  };
  auto match1 = [&](int i) -> bool { return canon(sl.bits(i)) == bits && sl.allowed(i); };
  // (the single values before the groups: every warp looks at them, so that no barrier is needed)
  const unsigned hm = __ballot_sync(0xffffffffu, lane < sl.head && match1(sl.i0 + lane));
  int want = nth;
  if (want < __popc(hm)) {
    if (threadIdx.x == 0) p.out_tokens[row] = sl.i0 + nth_bit(hm, want);
    return;
  }
  want -= __popc(hm);
  constexpr int U = 8;  // groups in flight per lane
  int turn = 0;
  for (int g0 = 0; g0 < sl.nv; g0 += kThreads * U, turn ^= 1) {
    const int g = g0 + warp * 32 * U + lane;
    uint4 v[U];
    unsigned m[U];
#pragma unroll
    for (int q = 0; q < U; ++q)
      if (g + 32 * q < sl.nv) v[q] = sl.group(g + 32 * q);
    int n = 0;
#pragma unroll
    for (int q = 0; q < U; ++q) {
      m[q] = g + 32 * q < sl.nv ? match8(v[q], g + 32 * q) : 0u;
      n += __popc(m[q]);
    }
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) sh.whits[turn][warp] = n;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) before = all;
      all += sh.whits[turn][w];
    }
    if (want >= all) {
      want -= all;
      continue;
    }
    want -= before;
    if (want < 0 || want >= n) return;  // another warp's
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int own = __popc(m[q]);
      const int here = __reduce_add_sync(0xffffffffu, own);
      if (want >= here) {
        want -= here;
        continue;
      }
      int inc = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int c = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += c;
      }
      if (want >= inc - own && want < inc) p.out_tokens[row] = sl.v0 + 8 * (g + 32 * q) + nth_bit(m[q], want - (inc - own));
      return;
    }
  }
  const unsigned tm = __ballot_sync(0xffffffffu, lane < sl.tail && match1(sl.t0 + lane));
  if (threadIdx.x == 0) p.out_tokens[row] = sl.t0 + nth_bit(tm, want);
}

// A row with values outside the main bins, by one CTA: four windows of the whole key space, counted
// again for each of the three sums (largest value and mass, kept mass, the draw).
__device__ __noinline__ void any_row(const SampleUniformParams& p, int row, Rules rule, double top_p, float u,
                                     int* hist, Shared& sh) {
  constexpr int kPer = kWindow / kThreads;
  const int tid = threadIdx.x;
  const Slice sl = make_slice(p, row, 0, 1);
  const int j0 = tid * kPer;
  auto at = [&](int i) -> int { return hist[j0 + i]; };
  auto count = [&](int win) {
    __syncthreads();
    for (int i = tid; i < kWindow; i += kThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < p.V; i += kThreads)
      if (sl.allowed(i)) count_window(sl.bits(i), win, hist);
    __syncthreads();
  };
  double mass = 0.0, em = 0.0, tm = 0.0;
  int n = 0, en = 0, tn = 0;
  auto prefix = [&](int win) {
    mass = 0.0;
    n = 0;
    for (int i = 0; i < kPer; ++i) {
      const int c = at(i);
      if (c > 0) mass += (double)c * exp_neg(rule.logw(bin_bits(j0 + i, win)));
      n += c;
    }
    __syncthreads();
    block_prefix(sh, 0, mass, n, em, en, tm, tn);
  };
  double z = 0.0;
  bool found = false;
  for (int win = 0; win < 4; ++win) {
    count(win);
    if (!found) {
      int first = kNone;
      for (int i = kPer - 1; i >= 0; --i)
        if (at(i) > 0) first = j0 + i;
      first = block_min(sh, 0, first);
      if (first == kNone) continue;
      found = true;
      rule.vmax = bf16_value(bin_bits(first, win));
    }
    prefix(win);
    z += tm;
  }
  rule.border = top_p < 1.0 ? top_p * z : INFINITY;
  double total = 0.0, bm = 0.0;
  long long bn = 0;
  for (int win = 0; win < 4; ++win) {
    count(win);
    prefix(win);
    const double kept = n > 0 ? walk(rule, at, j0, kPer, win, bm + em, bn + en, -1.0, nullptr, nullptr) : 0.0;
    __syncthreads();
    total += block_sum(sh, 1, kept);
    bm += tm;
    bn += tn;
  }
  const double target = (double)u * total;
  bm = 0.0;
  bn = 0;
  int bits = -1, place = 0;
  for (int win = 0; win < 4; ++win) {
    count(win);
    prefix(win);
    int b = -1, k = 0;
    if (n > 0 && (bn + en == 0 || bm + em <= target)) walk(rule, at, j0, kPer, win, bm + em, bn + en, target, &b, &k);
    const int last = -block_min(sh, 1, b >= 0 ? -tid : kNone);  // the last thread with a kept value
    if (last >= 0) {
      if (tid == last) {
        sh.r_bits = b;
        sh.r_rank = k;
      }
      __syncthreads();
      bits = sh.r_bits;
      place = sh.r_rank;
    }
    bm += tm;
    bn += tn;
  }
  find_token(p, row, sl, sh, bits, place);
  if (tid == 0 && p.out_logprob) p.out_logprob[row] = (float)(rule.logw(bits) - log(total));
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
  const int tid = threadIdx.x, lane = tid & 31;
  auto peer = [&](int r) -> Shared* {
    if constexpr (C == 1) return &sh;
    else return cl.map_shared_rank(&sh, r);
  };
  const Slice sl = make_slice(p, row, rank, C);
  const float tf = p.temperature ? p.temperature[row] : 0.f;
  constexpr int U = 4;  // 16-byte groups in flight

  if (!(tf > 0.f)) {  // greedy: the largest value (packed maxima, which pass over NaN), then its first place
    const __nv_bfloat162 none = __floats2bfloat162_rn(-INFINITY, -INFINITY);
    __nv_bfloat162 best = none;
    auto one = [&](int i) {
      if (sl.allowed(i)) best = __hmax2(best, __halves2bfloat162(sl.row[i], none.x));
    };
    if (tid < sl.head) one(sl.i0 + tid);
    if (tid < sl.tail) one(sl.t0 + tid);
    for (int g0 = tid; g0 < sl.nv; g0 += kThreads * U) {
      uint4 v[U];
      unsigned allow[U];  // (loaded with the values: one wait for both)
#pragma unroll
      for (int q = 0; q < U; ++q)
        if (g0 + q * kThreads < sl.nv) {
          v[q] = sl.group(g0 + q * kThreads);
          allow[q] = sl.allowed8(sl.v0 + 8 * (g0 + q * kThreads));
        }
#pragma unroll
      for (int q = 0; q < U; ++q) {
        const int g = g0 + q * kThreads;
        if (g >= sl.nv) break;
        const unsigned w[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
        const unsigned ok = allow[q];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          unsigned x = w[j];
          if (ok != 0xffu) {  // disallowed: -inf
            if (!((ok >> (2 * j)) & 1u)) x = (x & 0xffff0000u) | 0xff80u;
            if (!((ok >> (2 * j)) & 2u)) x = (x & 0xffffu) | 0xff800000u;
          }
          best = __hmax2(best, *reinterpret_cast<const __nv_bfloat162*>(&x));
        }
      }
    }
    float top = fmaxf(__low2float(best), __high2float(best));
    top = top == 0.f ? 0.f : top == top ? top : -INFINITY;  // (zeros of both signs are one value: one key)
    const unsigned tb = __float_as_uint(top);
    // bf16 keys are the upper halves of fp32 keys: a minimum of complements is a maximum
    int key = -(int)(((tb & 0x80000000u) ? ~tb : (tb | 0x80000000u)) >> 16);
    key = block_min(sh, 0, key);
    if constexpr (C > 1) {
      if (tid == 0) sh.in[0].first = key;
      cl.sync();  // (also: a peer's memory may be touched only once the peer has started)
      int r = 0, low = peer(0)->in[0].first;
#pragma unroll
      for (int q = 1; q < C; ++q) {
        const int k = peer(q)->in[0].first;
        if (k < low) {
          low = k;
          r = q;
        }
      }
      cl.sync();  // every peer has read this CTA's key
      if (r != rank) return;
    }
    const int k16 = -key;
    const int bits = (k16 & 0x8000) ? (k16 ^ 0x8000) : (~k16 & 0xffff);
    if (bits == 0xff80) {  // no token
      if (tid == 0) {
        p.out_tokens[row] = -1;
        if (p.out_logprob) p.out_logprob[row] = -INFINITY;
      }
      return;
    }
    if (tid == 0 && p.out_logprob) p.out_logprob[row] = 0.f;
    find_token(p, row, sl, sh, canon((unsigned)bits), 0);
    return;
  }

  // ---- histogram of the slice
  for (int i = tid; i < kHist / 4; i += kThreads) reinterpret_cast<int4*>(hist)[i] = make_int4(0, 0, 0, 0);
  if (tid == 0) {
    sh.odd = 0;
    sh.edge = kThreads;
  }
  __syncthreads();
  {
    bool inside = true;
    if (tid < sl.head && sl.allowed(sl.i0 + tid)) inside &= count_main(sl.bits(sl.i0 + tid), hist);
    if (tid < sl.tail && sl.allowed(sl.t0 + tid)) inside &= count_main(sl.bits(sl.t0 + tid), hist);
    for (int g0 = tid; g0 < sl.nv; g0 += kThreads * U) {
      uint4 v[U];
      unsigned allow[U];  // (loaded with the values: one wait for both)
#pragma unroll
      for (int q = 0; q < U; ++q)
        if (g0 + q * kThreads < sl.nv) {
          v[q] = sl.group(g0 + q * kThreads);
          allow[q] = sl.allowed8(sl.v0 + 8 * (g0 + q * kThreads));
        }
#pragma unroll
      for (int q = 0; q < U; ++q) {
        const int g = g0 + q * kThreads;
        if (g >= sl.nv) break;
        const unsigned w[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
        const unsigned ok = allow[q];
        if (ok == 0u) continue;
        const bool plain = main_word(w[0]) && main_word(w[1]) && main_word(w[2]) && main_word(w[3]);
        if (plain && ok == 0xffu) {
#pragma unroll
          for (int j = 0; j < 4; ++j) count_word<true>(w[j], 3u, hist);
        } else if (plain) {
#pragma unroll
          for (int j = 0; j < 4; ++j) count_word<false>(w[j], ok >> (2 * j), hist);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if ((ok >> j) & 1u) inside &= count_main((w[j >> 1] >> (16 * (j & 1))) & 0xffffu, hist);
        }
      }
    }
    if (!inside) sh.odd = 1;
  }
  float u = p.uniforms[row];
  u = u > 0.f ? fminf(u, 1.f) : 0.f;
  const double top_p = p.top_p ? (double)p.top_p[row] : 1.0;
  const int top_k = p.top_k ? p.top_k[row] : 0;
  Rules rule;
  rule.inv_t = 1.0 / (double)tf;
  rule.min_p = p.min_p ? (double)p.min_p[row] : 0.0;
  rule.border = INFINITY;
  rule.K = top_k > 0 ? top_k : (long long)kNone;
  rule.vmax = 0.0;
  row_sync<C>(cl);
  // ---- (C > 1) the row's counts of this CTA's share of the signed values (a block of the counters, see
  // main_at), and of zero
  constexpr int kShare = 2 * kMagN / C;
  const int block = main_at(bin_bits(nth_bin(rank * kShare), -1)) & ~(kShare - 1);
  int* own = hist + kHist;
  if constexpr (C > 1) {
    int c0 = 0;
    if (tid < C) c0 = cl.map_shared_rank(hist, tid)[2 * kMagN];
#pragma unroll
    for (int a = tid; a < kShare / 4; a += kThreads) {
      int4 c = make_int4(0, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < C; ++r) {
        const int4 h = reinterpret_cast<const int4*>(cl.map_shared_rank(hist, r) + block)[a];
        c.x += h.x;
        c.y += h.y;
        c.z += h.z;
        c.w += h.w;
      }
      reinterpret_cast<int4*>(own)[a] = c;
    }
    if (tid < 32) {
      c0 = __reduce_add_sync(0xffffffffu, c0);
      if (tid == 0) own[kShare] = c0;
    }
  }
  if (__syncthreads_or(tid < C && peer(tid)->odd != 0)) {
    if constexpr (C > 1) cl.sync();  // every peer has read the flags: rank 0 may reuse its memory
    if (rank == 0) any_row(p, row, rule, top_p, u, hist, sh);
    return;
  }

  // ---- the non-empty bins of this CTA's share (1/C of the signed values; zero goes with the smallest
  // positive ones), as a list in descending order of value, so that afterwards the exponentials (a few
  // hundred cycles each) spread evenly over the threads. A warp takes 1/16 of the share, its lanes
  // neighbouring bins, 16 bytes of counters at a time, first to count, then to place.
  constexpr int kChunks = kShare / (128 * kWarps);
  unsigned short* list = reinterpret_cast<unsigned short*>(own + (C > 1 ? kShare + 4 : 0));
  auto count = [&](int j) -> int {
    const int a = main_at(bin_bits(j, -1));
    if constexpr (C > 1) return own[j == kMagN ? kShare : a - block];
    else return hist[a];
  };
  int len;
  {
    const int i0 = (rank * kWarps + (tid >> 5)) * kChunks * 128;
    const bool with_zero = i0 + kChunks * 128 == kMagN && count(kMagN) > 0;
    // the warp's counters are consecutive (downwards for positive values, upwards for negative ones): a
    // lane takes four neighbours at a time; flags: bit 4 k + b = its b-th bin of chunk k is not empty
    const bool up = i0 >= kMagN;
    const int* c0 = (C > 1 ? own - block : hist) + main_at(bin_bits(nth_bin(i0), -1)) + (up ? 4 * lane : -4 * lane - 3);
    unsigned flags = 0;
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int4 v = *reinterpret_cast<const int4*>(c0 + (up ? 128 * k : -128 * k));
      const unsigned f = (v.x > 0 ? 1u : 0u) | (v.y > 0 ? 2u : 0u) | (v.z > 0 ? 4u : 0u) | (v.w > 0 ? 8u : 0u);
      flags |= (up ? f : __brev(f) >> 28) << (4 * k);
    }
    const int filled = __reduce_add_sync(0xffffffffu, __popc(flags)) + with_zero;
    if (lane == 0) sh.cnt[tid >> 5] = filled;
    __syncthreads();
    int at = 0;
    len = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w == (tid >> 5)) at = len;
      len += sh.cnt[w];
    }
    if (filled > 0) {
      const unsigned below = (1u << lane) - 1u;
      const int j0 = nth_bin(i0) + 4 * lane;
#pragma unroll
      for (int k = 0; k < kChunks; ++k) {
        const unsigned f = (flags >> (4 * k)) & 15u;
        unsigned m[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) m[b] = __ballot_sync(0xffffffffu, (f >> b) & 1u);
        if ((m[0] | m[1] | m[2] | m[3]) == 0u) continue;
        int to = at, next = at;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          to += __popc(m[b] & below);
          next += __popc(m[b]);
        }
#pragma unroll
        for (int b = 0; b < 4; ++b)
          if ((f >> b) & 1u) list[to++] = (unsigned short)(j0 + 128 * k + b);
        at = next;
      }
      if (with_zero && lane == 0) list[at] = (unsigned short)kMagN;
    }
  }
  __syncthreads();
  auto bin = [&](int e) -> int { return (int)list[e]; };
  int first = len > 0 ? bin(0) : kNone;
  const int per = (len + kThreads - 1) / kThreads;
  const int e0 = min(len, tid * per), e1 = min(len, e0 + per);

  // ---- masses relative to the CTA's largest value, exchanged and put on the row's scale
  double mass = 0.0, w_hi = 0.0, w_lo = 0.0;
  int n = 0;
  rule.vmax = first != kNone ? bf16_value(bin_bits(first, -1)) : 0.0;
  for (int e = e0; e < e1; e += 2) {
    const int ja = bin(e), jb = e + 1 < e1 ? bin(e + 1) : ja;
    const int ca = count(ja), cb = e + 1 < e1 ? count(jb) : 0;
    const double wa = exp_neg(rule.logw(bin_bits(ja, -1))), wb = exp_neg(rule.logw(bin_bits(jb, -1)));
    if (e == e0) w_hi = wa;
    w_lo = wb;
    n += ca + cb;
    mass += (double)ca * wa + (double)cb * wb;
  }
  double m0, tm;
  int en, tn;
  block_prefix(sh, 1, mass, n, m0, en, tm, tn);
  double z = tm;
  long long n0 = en;
  if constexpr (C > 1) {
    if (tid < C) {
      Shared* o = peer(tid);
      o->in[rank].mass = tm;
      o->in[rank].cnt = tn;
      o->in[rank].first = first;
    }
    cl.sync();
    int row_first = kNone;
#pragma unroll
    for (int r = 0; r < C; ++r) row_first = min(row_first, sh.in[r].first);
    if (row_first != kNone) rule.vmax = bf16_value(bin_bits(row_first, -1));
    if (tid < C) {
      const int f = sh.in[tid].first;
      sh.scale[tid] = f != kNone ? exp_neg(rule.logw(bin_bits(f, -1))) : 0.0;
    }
    __syncthreads();
    z = 0.0;
    long long before = 0;
    double base = 0.0;
#pragma unroll
    for (int r = 0; r < C; ++r) {
      if (r == rank) {
        base = z;
        n0 += before;
      }
      z += sh.in[r].mass * sh.scale[r];
      before += sh.in[r].cnt;
    }
    const double scale = sh.scale[rank];
    mass *= scale;
    w_hi *= scale;
    w_lo *= scale;
    m0 = base + m0 * scale;
    first = row_first;
  }
  if (first == kNone) {  // no token at all (the same in every CTA of the row)
    if (rank == 0 && tid == 0) {
      p.out_tokens[row] = -1;
      if (p.out_logprob) p.out_logprob[row] = -INFINITY;
    }
    if constexpr (C > 1) cl.sync();
    return;
  }
  rule.border = top_p < 1.0 ? top_p * z : INFINITY;

  // ---- kept mass: all of a thread's entries, none, or, in the one thread at the end of the kept
  // prefix, a part (every warp works that part out)
  const bool any = n > 0 && (n0 == 0 || (n0 < rule.K && m0 < rule.border && w_hi >= rule.min_p));
  const bool whole = any && n0 + n <= rule.K && m0 + mass < rule.border && w_lo >= rule.min_p;
  // (rounding may let a later thread think that it is the one: the first counts)
  const unsigned ends = __ballot_sync(0xffffffffu, any && !whole);
  if (ends != 0 && lane == __ffs(ends) - 1) {
    atomicMin(&sh.edge, tid);
    sh.end[tid >> 5] = {e0, e1 - e0, n0, m0};
  }
  double cta_kept = block_sum(sh, 0, whole ? mass : 0.0);
  const int edge = sh.edge;
  if (edge < kThreads) {
    const auto& end = sh.end[edge >> 5];
    cta_kept += warp_walk(rule, bin, count, end.first, end.n, end.m0, end.n0, -1.0, nullptr, nullptr);
  }
  double total = cta_kept;
  int sel = 0;  // CTA that holds the target
  if constexpr (C > 1) {
    if (tid < C) peer(tid)->in[rank].kept = cta_kept;
    cl.sync();
    total = 0.0;
#pragma unroll
    for (int r = 0; r < C; ++r) total += sh.in[r].kept;
  }
  const double target = (double)u * total;
  if constexpr (C > 1) {  // the last CTA with kept tokens whose preceding kept mass is <= target
    double before = 0.0;
#pragma unroll
    for (int r = 0; r < C; ++r) {
      const double k = sh.in[r].kept;
      if (k > 0.0 && (before <= target || before == 0.0)) sel = r;
      before += k;
    }
  }

  // ---- the draw: the last thread of that CTA with kept tokens that starts at or below the target (or
  // the first, should rounding put that start above)
  const bool has = rank == sel && any;
  const int lead = block_min(sh, 1, has ? tid : kNone);
  const int head = -block_min(sh, 0, has && (m0 <= target || tid == lead) ? -tid : kNone);
  if (rank == sel && (tid >> 5) == (head >> 5)) {
    int b = -1, k = 0;
    const int src = head & 31;
    warp_walk(rule, bin, count, __shfl_sync(0xffffffffu, e0, src), __shfl_sync(0xffffffffu, e1 - e0, src),
              __shfl_sync(0xffffffffu, m0, src), __shfl_sync(0xffffffffu, n0, src), target, &b, &k);
    if (lane < C) {
      peer(lane)->r_bits = b;
      peer(lane)->r_rank = k;
    }
  }
  row_sync<C>(cl);
  const int bits = sh.r_bits;
  int nth = sh.r_rank;
  // ---- the slice that holds the nth token of this value: its counts are still in the histograms
  if constexpr (C > 1) {
    const int c = lane < rank ? cl.map_shared_rank(hist, lane)[main_at(bits)] : 0;
    nth -= __reduce_add_sync(0xffffffffu, c);
    if (nth >= 0 && nth < hist[main_at(bits)]) find_token(p, row, sl, sh, bits, nth);
  } else {
    find_token(p, row, sl, sh, bits, nth);
  }
  if (rank == sel && tid == 0 && p.out_logprob) p.out_logprob[row] = (float)(rule.logw(bits) - log(total));
  if constexpr (C > 1) cl.sync();  // peers may still read this CTA's shared memory
}

template <int C>
cudaError_t launch_c(const SampleUniformParams& p, cudaStream_t s) {
  // histogram, the row's counts of the CTA's share (C > 1), list of its non-empty bins
  constexpr size_t smem = (size_t)(kHist + (C > 1 ? 2 * kMagN / C + 4 : 0)) * sizeof(int) + (size_t)(2 * kMagN / C + 8) * 2;
  cudaError_t e = allow_smem(sample_uniform_kernel<C>, (int)smem);
  if (e != cudaSuccess) return e;
  SQ_LAUNCH(sample_uniform_kernel<C>, dim3(p.B, 1, C), dim3(kThreads), smem, s, C, p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t sample_uniform_launch(const SampleUniformParams& p, int num_sms, cudaStream_t s) {
  if (p.B == 0) return cudaSuccess;
  if (p.V <= 0) return cudaErrorInvalidValue;
  // CTAs per row. A cluster counts its row faster and pays for it with exchanges: up to 32000 values one
  // CTA is as fast or faster at any batch (1 row of 32000: 13.2 us against 13.9, 13.1, 13.9 with 2, 4, 8;
  // 64 rows: 13.7 against 14.3, 20.3, 42.2). Of 152064 values, us with 1, 2, 4, 8 CTAs: 1 row 23, 19, 17,
  // 16; 8 rows 30, 23, 19, 17; 16 rows 30, 23, 18, 20; 64 rows 30, 23, 26, 47; 100 rows 31, 42, 43, 75 (two
  // CTAs of two do not fit an SM). Where between the two sizes the change pays most was not measured.
  int c = 1;
  if (p.V > 65536) c = 16 * p.B <= num_sms ? 8 : 8 * p.B <= num_sms ? 4 : 2 * p.B <= num_sms ? 2 : 1;
  switch (c) {
    case 8: return launch_c<8>(p, s);
    case 4: return launch_c<4>(p, s);
    case 2: return launch_c<2>(p, s);
    default: return launch_c<1>(p, s);
  }
}

}  // namespace sq
