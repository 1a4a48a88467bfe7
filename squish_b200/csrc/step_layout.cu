// step_layout.cu — block tables, slot map and attention tiles of a step from its request lengths.
//
//   q_start = exclusive prefix sum of q            kv[b] = ctx[b] + q[b]
//   new pages of b = ceil(kv / page) - ceil(ctx / page), taken from the free list in sequence order
//   position(t) = ctx[b] + t - q_start[b]          slot(t) = page(position / page) * page + rest
//   attention tiles: ceil(q / tile) per sequence, in sequence order
//
// Every block scans the lengths of all sequences itself (8 bytes each, from L2) and then writes its
// share of the token, tile and page rows, found by binary search in the prefixes in shared memory.
// A sequence whose tokens do not all fit rests (kv_len of what it had, tiles that are padding).
// No block needs another's result: the page of a new token comes from the free list, not from the
// table entry that another block may be writing. So the step is one launch with no grid-wide wait.
// What bounds it is latency: launch, lengths, scan, search, page, slot (64 sequences: 3.5 us for 3 KB;
// 1000 sequences, 250000 tokens: 6.8 us for 3.2 MB).
#include "kernels.h"
#include "launch.cuh"
#include "sm100.cuh"
#include "step_ops.h"

namespace sq {

namespace {

constexpr int kThreads = 256;
constexpr unsigned kSat = 1u << 30;  // prefixes saturate here: sums of any valid lengths stay in 32 bits

__device__ __forceinline__ unsigned sat_add(unsigned a, unsigned b) { return min(a + b, kSat); }

// number of entries of the non-decreasing pre[1..n] that are <= v
__device__ __forceinline__ int upper(const unsigned* pre, int n, unsigned v) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid + 1] <= v) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

template <int V>
__global__ void __launch_bounds__(kThreads) step_layout_kernel(const StepLayoutParams p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ unsigned sh[];
  const int B = p.B, ps = p.page_size;
  unsigned* qs = sh;             // [B + 1] tokens before sequence b
  unsigned* pg = qs + B + 1;     // [B + 1] new pages before sequence b
  unsigned* ts = pg + B + 1;     // [B + 1] tiles before sequence b
  int* ctx = reinterpret_cast<int*>(ts + B + 1);  // [B]
  __shared__ unsigned wsum[3][kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (B + kThreads - 1) / kThreads;
  const int b0 = min(B, tid * per), b1 = min(B, b0 + per);
  bool bad = false;
  unsigned s0 = 0, s1 = 0, s2 = 0;
  for (int b = b0; b < b1; ++b) {
    int c = p.ctx_len[b], q = p.q_len[b];
    if (c < 0 || c >= (int)kSat || q < 0 || q > (int)kSat) {  // not a length: the sequence counts as resting
      bad = true;
      c = (c < 0 || c >= (int)kSat) ? 0 : c;
      q = 0;
    }
    ctx[b] = c;
    const unsigned have = (unsigned)(c + ps - 1) / (unsigned)ps;
    const unsigned need = ((unsigned)c + (unsigned)q + (unsigned)(ps - 1)) / (unsigned)ps - have;
    qs[b + 1] = s0 = sat_add(s0, q);
    pg[b + 1] = s1 = sat_add(s1, need);
    ts[b + 1] = s2 = sat_add(s2, (unsigned)(q + p.tile - 1) / (unsigned)p.tile);
  }
  // exclusive prefix of the threads' sums: within the warp, then over the warps
  unsigned i0 = s0, i1 = s1, i2 = s2;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned a = __shfl_up_sync(0xffffffffu, i0, o), b = __shfl_up_sync(0xffffffffu, i1, o),
                   c = __shfl_up_sync(0xffffffffu, i2, o);
    if (lane >= o) {
      i0 = sat_add(i0, a);
      i1 = sat_add(i1, b);
      i2 = sat_add(i2, c);
    }
  }
  if (lane == 31) {
    wsum[0][warp] = i0;
    wsum[1][warp] = i1;
    wsum[2][warp] = i2;
  }
  __syncthreads();
  unsigned e0 = __shfl_up_sync(0xffffffffu, i0, 1), e1 = __shfl_up_sync(0xffffffffu, i1, 1),
           e2 = __shfl_up_sync(0xffffffffu, i2, 1);
  if (lane == 0) e0 = e1 = e2 = 0;
  for (int w = 0; w < warp; ++w) {
    e0 = sat_add(e0, wsum[0][w]);
    e1 = sat_add(e1, wsum[1][w]);
    e2 = sat_add(e2, wsum[2][w]);
  }
  for (int b = b0; b < b1; ++b) {
    qs[b + 1] = sat_add(qs[b + 1], e0);
    pg[b + 1] = sat_add(pg[b + 1], e1);
    ts[b + 1] = sat_add(ts[b + 1], e2);
  }
  if (tid == 0) qs[0] = pg[0] = ts[0] = 0;
  __syncthreads();
  const int T = (int)qs[B], P = (int)pg[B], NT = (int)ts[B];
  // Rows, pages and table columns for all of a sequence's tokens? What reads the cache goes by kv_len and
  // the tiles: past a missing page lies what another request stored, past the row's width another row.
  const unsigned held = (unsigned)min((long long)p.bt_width * ps, 0xffffffffll);  // tokens of a full table row
  auto fits = [&](int b) -> bool {
    return qs[b + 1] <= (unsigned)p.token_cap && (pg[b + 1] == pg[b] || pg[b + 1] <= (unsigned)p.n_free) &&
           (unsigned)ctx[b] + (qs[b + 1] - qs[b]) <= held;
  };
  if (blockIdx.x == 0) {
    if (T > p.token_cap || NT > p.tile_cap || P > p.n_free) bad = true;
    for (int b = tid; b <= B; b += kThreads) {
      p.q_start[b] = (int)qs[b];
      if (b == B) break;
      const int q = (int)(qs[b + 1] - qs[b]);
      const bool whole = fits(b);
      if ((unsigned)ctx[b] > held) bad = true;
      p.kv_len[b] = whole ? ctx[b] + q : (int)min((unsigned)ctx[b], held);
      p.last_row[b] = whole && q > 0 ? (int)qs[b + 1] - 1 : -1;
    }
    if (tid == 0) {
      p.totals[0] = T;
      p.totals[1] = P;
      p.totals[2] = NT;
    }
  }
  const int stride = gridDim.x * kThreads, first = blockIdx.x * kThreads + tid;
  // V consecutive tokens per thread: one search, one page lookup while they share a page
  for (int qv = first; qv < (p.token_cap + V - 1) / V; qv += stride) {
    const int t0 = V * qv;
    int pos[V], slot[V], sq[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      pos[j] = 0;
      slot[j] = sq[j] = -1;
    }
    if (t0 < T) {
      int seq = upper(qs, B, (unsigned)t0);
      int c = ctx[seq], pi = -1, page = -1;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int t = t0 + j;
        if (t >= T || t >= p.token_cap) break;
        while (t >= (int)qs[seq + 1]) {  // (the next sequence with tokens: t < T, so there is one)
          ++seq;
          c = ctx[seq];
          pi = -1;
        }
        pos[j] = c + (t - (int)qs[seq]);
        sq[j] = seq;
        if (pi < 0 || pos[j] >= (pi + 1) * ps) {
          pi = pos[j] / ps;
          const int have = (c + ps - 1) / ps;
          page = -1;
          if (pi >= p.bt_width) {
            bad = true;
          } else if (pi < have) {
            page = p.block_tables[(size_t)seq * p.bt_stride + pi];
          } else {
            const int f = (int)pg[seq] + (pi - have);
            if (f < p.n_free) page = p.free_pages[f];
          }
        }
        const long long sl = (long long)page * ps + (pos[j] - pi * ps);
        if (page >= 0) {  // (a page given back reads -1: nothing is stored)
          if (sl <= 0x7fffffffll) slot[j] = (int)sl;
          else bad = true;
        }
      }
    }
    if constexpr (V == 4) {  // 16-byte stores: the rows are padded to whole groups of four
      reinterpret_cast<int4*>(p.positions)[qv] = make_int4(pos[0], pos[1], pos[2], pos[3]);
      reinterpret_cast<int4*>(p.slots)[qv] = make_int4(slot[0], slot[1], slot[2], slot[3]);
      reinterpret_cast<int4*>(p.token_seq)[qv] = make_int4(sq[0], sq[1], sq[2], sq[3]);
    } else {
      p.positions[qv] = pos[0];
      p.slots[qv] = slot[0];
      p.token_seq[qv] = sq[0];
    }
  }
  for (int i = first; i < p.tile_cap; i += stride) {
    int seq = 0, q0 = kLayoutPadQ0;
    if (i < NT) {
      const int b = upper(ts, B, (unsigned)i);
      if (fits(b)) {
        seq = b;
        q0 = (i - (int)ts[b]) * p.tile;
      }
    }
    p.tile_seq[i] = seq;
    p.tile_q0[i] = q0;
  }
  for (int i = first; i < min(P, p.n_free); i += stride) {
    const int seq = upper(pg, B, (unsigned)i);
    const int pi = (ctx[seq] + ps - 1) / ps + (i - (int)pg[seq]);
    if (pi < p.bt_width) p.block_tables[(size_t)seq * p.bt_stride + pi] = p.free_pages[i];
    else bad = true;
  }
  if (bad) atomicCAS(p.status, 0, SQ_ERR_BOUNDS);
}

}  // namespace

cudaError_t step_layout_launch(const StepLayoutParams& p, int num_sms, cudaStream_t s) {
  if (p.B <= 0 || p.B > kLayoutMaxSeqs || p.page_size <= 0 || p.tile <= 0) return cudaErrorInvalidValue;
  const size_t smem = (size_t)(4 * p.B + 3) * sizeof(int);
  // One token per thread while a wave of blocks holds them (64 sequences, 64 tokens: 3.5 us against
  // 4.9), four from there on (1000 sequences, 250000 tokens: 6.8 us against 8.4).
  const int v = p.token_cap > 65536 ? 4 : 1;
  auto* kern = v == 4 ? step_layout_kernel<4> : step_layout_kernel<1>;
  // (the kernel's static arrays count towards the 48 KB that need no permission: 3066 to 3071 sequences
  // stay below it with their prefixes alone)
  if (smem > 47 * 1024) {
    const cudaError_t e = allow_smem(kern, 4 * (4 * kLayoutMaxSeqs + 3));
    if (e != cudaSuccess) return e;
  }
  const int rows = (p.token_cap + v - 1) / v > p.tile_cap ? (p.token_cap + v - 1) / v : p.tile_cap;
  int blocks = (rows + kThreads - 1) / kThreads;
  if (blocks > 4 * num_sms) blocks = 4 * num_sms;
  if (blocks < 1) blocks = 1;
  SQ_LAUNCH(kern, dim3(blocks), dim3(kThreads), smem, s, 1, p);
  return cudaGetLastError();
}

}  // namespace sq
